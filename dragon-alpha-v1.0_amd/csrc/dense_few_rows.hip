// The dense product for few rows of X or little work: no copy of an operand, one launch (two where a long reduction of few workgroups
// is cut), as many bytes in flight as the device takes. A single row reads W once and is bound by that: 1 x 4096 x 4096 bf16 8.1 us, 4.2 TB/s; a gated pair 1 x 2048 x 8192
// 12.4 us, 5.4 TB/s. More rows are bound by what a compute unit loads (35 to 40 bytes a nanosecond, whatever is in flight).
//
// A workgroup of eight wavefronts computes 16 columns of the output (16 rows of W) for 16, 32 or 64 rows of X; its wavefronts
// share the reduction in pieces of 256 bytes of every row. Both operands go straight from memory into the MFMA registers: a
// lane holds 16 bytes of one row of W and of one row of X at the same k. bf16: v_mfma_f32_16x16x32_bf16, eight k a lane;
// fp32: v_mfma_f32_16x16x4_f32, component s of the lane's four k in the s-th MFMA - plain fp32 products. Rows of X beyond
// the last are the last once more, their results not stored. The partial sums are added through LDS in a fixed order.
// At most four rows of X: four columns a workgroup instead of 16, the MFMA's 16 rows and columns being four pieces of the
// reduction times four (only the products of equal pieces are read out): four times as many workgroups, each with a
// quarter of the reduction's length in turns (1 x 8192 x 1024 of bf16: 11.4 -> 5.4 us).
// Rows may begin at any element and K may be any number.
#include "dense_direct.hpp"

#include <algorithm>

namespace alpha {

namespace {

constexpr int FEW_WAVES = 8;

}  // namespace

// C: columns of a workgroup, 16, or 4 for at most four rows. MB: blocks of 16 rows.
template <typename T, bool ODD, bool GATED, int MB, int C>
__global__ __launch_bounds__(FEW_WAVES * 64, !ODD && !GATED && MB == 4 ? 4 : 2) void dense_few_rows_kernel(const DenseFewRows a)
{
    typedef typename FewVec<T>::type vec;
    constexpr int V = 16 / sizeof(T), CHUNK = 4 * V, GROUPS = 16 / C;         // k of a lane, of a wavefront's load of a row
    constexpr int PIECE = 4 * CHUNK, SPAN = GROUPS * PIECE;                   // of a row at a time, of a wavefront's turn
    constexpr int G = GATED ? 2 : 1;
    static_assert(C == 16 || MB == 1, "few columns are for few rows");
    __shared__ floatx4 part[FEW_WAVES][G * MB][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, q = lane >> 4;
    const int n0 = blockIdx.x * C, n = n0 + l16 % C < a.N ? n0 + l16 % C : a.N - 1, m0 = blockIdx.y * (MB * 16);
    const T *w[G], *x[MB];
    w[0] = static_cast<const T *>(a.W) + n * a.ldW;
    if constexpr (GATED) w[1] = static_cast<const T *>(a.W2) + n * a.ldW2;
#pragma unroll
    for (int b = 0; b < MB; b++) {
        const int m = m0 + b * 16 + l16 % C;
        x[b] = static_cast<const T *>(a.X) + (m < a.M ? m : a.M - 1) * a.ldX;
    }
    floatx4 acc[G][MB];
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int b = 0; b < MB; b++) acc[g][b] = floatx4{0.f, 0.f, 0.f, 0.f};

    // Every workgroup starts at another place of the reduction: rows are often a power of two apart, and workgroups that
    // all read the same k at a time would all ask the same few channels of the memory.
    // (bf16, rows that begin with a word: the last load of a row ends with the word of its last element)
    const int end = sizeof(T) == 2 && !ODD ? (a.K + 1) & ~1 : a.K, last = end - V;
    const int turns = a.K < V ? 0 : (a.K + FEW_WAVES * SPAN - 1) / (FEW_WAVES * SPAN);
    const int from = blockIdx.z * a.per, to = from + a.per < turns ? from + a.per : turns, count = to - from;
    int turn = count > 0 ? from + (int)(blockIdx.x % count) : 0;
    for (int t = 0; t < count; t++) {
        const int k0 = (turn * FEW_WAVES + wave) * SPAN, k = k0 + l16 / C * PIECE;
        if (k0 < a.K) {
            vec vw[G][4], vx[MB][4];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int at = k + c * CHUNK + q * V;
#pragma unroll
                for (int g = 0; g < G; g++) vw[g][c] = few_load<ODD>(w[g], at < last ? at : last);
            }
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int at = k + c * CHUNK + q * V;
#pragma unroll
                for (int b = 0; b < MB; b++) vx[b][c] = few_load<ODD>(x[b], at < last ? at : last);
            }
            const bool edge = k0 + SPAN > a.K;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                if (edge) {
#pragma unroll
                    for (int g = 0; g < G; g++) vw[g][c] = few_at_edge<T, ODD>(vw[g][c], k + c * CHUNK + q * V, end, a.K);
#pragma unroll
                    for (int b = 0; b < MB; b++) vx[b][c] = few_at_edge<T, ODD>(vx[b][c], k + c * CHUNK + q * V, end, a.K);
                }
#pragma unroll
                for (int g = 0; g < G; g++)
#pragma unroll
                    for (int b = 0; b < MB; b++) acc[g][b] = few_multiply(vw[g][c], vx[b][c], acc[g][b]);
            }
        }
        turn = turn + 1 == to ? from : turn + 1;
    }

    if (a.K < V && wave == 0) {   // less than one load: element by element, zeros behind and in the other lanes' pieces
        vec vw[G], vx[MB];
#pragma unroll
        for (int e = 0; e < V; e++) {
            const bool there = e < a.K && q == 0 && l16 < C;
#pragma unroll
            for (int g = 0; g < G; g++) vw[g][e] = there ? w[g][e] : (T)0.f;
#pragma unroll
            for (int b = 0; b < MB; b++) vx[b][e] = there ? x[b][e] : (T)0.f;
        }
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
            for (int b = 0; b < MB; b++) acc[g][b] = few_multiply(vw[g], vx[b], acc[g][b]);
    }
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int b = 0; b < MB; b++) part[wave][g * MB + b][lane] = acc[g][b];
    __syncthreads();
    // Lane (l16, q) of an MFMA result holds columns 4 q .. 4 q + 3 of row l16. C = 4: the sums of piece g are the columns
    // and rows 4 g .. 4 g + 3.
    for (int t = threadIdx.x; t < MB * 16 * C; t += FEW_WAVES * 64) {
        const int b = t / (16 * C), col = t % C, row = t / C % 16, m = m0 + b * 16 + row;
        if (row >= (C == 16 ? 16 : C) || m >= a.M || n0 + col >= a.N) continue;
        float v[1] = {0.f}, u[1] = {0.f};
#pragma unroll
        for (int s = 0; s < FEW_WAVES; s++)
#pragma unroll
            for (int g = 0; g < GROUPS; g++) {
                const int at = ((col + g * C) >> 2) * 16 + row + g * C;
                v[0] += reinterpret_cast<const float *>(&part[s][b][at])[col & 3];
                if constexpr (GATED) u[0] += reinterpret_cast<const float *>(&part[s][(GATED ? MB : 0) + b][at])[col & 3];
            }
        if (a.cuts > 1) {
            const long columns = (a.N + 3) & ~3;
            float *to = a.pieces + ((long)blockIdx.z * G * a.M + m) * columns + n0 + col;
            to[0] = v[0];
            if constexpr (GATED) to[a.M * columns] = u[0];
            continue;
        }
        if constexpr (GATED) dense_finish_gated<T, 1, false>(a.ep, v, u, m, n0 + col);
        else dense_finish<T, 1, true, false>(a.ep, v, m, n0 + col);
    }
}

// Adds the pieces of a cut reduction in their order: four columns a thread.
template <typename T, bool GATED>
__global__ __launch_bounds__(256) void dense_few_sum_kernel(const DenseFewRows a, FastDiv by_row)
{
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    const long m = fdiv((uint32_t)i, by_row), columns = (a.N + 3) & ~3;
    if (m >= a.M) return;
    const int n = (int)(i - m * by_row.d) * 4;
    constexpr int G = GATED ? 2 : 1;
    float v[G][4];
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int e = 0; e < 4; e++) v[g][e] = 0.f;
#pragma unroll 4
    for (int p = 0; p < a.cuts; p++) {
#pragma unroll
        for (int g = 0; g < G; g++) {
            // (columns behind the last are not written, and not used)
            const floatx4 t = quad_load(a.pieces + (((long)p * G + g) * a.M + m) * columns + n);
#pragma unroll
            for (int e = 0; e < 4; e++) v[g][e] += t[e];
        }
    }
    const int left = a.N - n < 4 ? a.N - n : 4;
    if constexpr (GATED) {
        if (a.ep.vec && left == 4) dense_finish_gated<T, 4, true>(a.ep, v[0], v[1], m, n);
        else dense_finish_gated<T, 4, false>(a.ep, v[0], v[1], m, n, left);
    } else {
        if (a.ep.vec && left == 4) dense_finish<T, 4, true, true>(a.ep, v[0], m, n);
        else dense_finish<T, 4, true, false>(a.ep, v[0], m, n, left);
    }
}

namespace {

// Four columns a workgroup or 16, for at most four rows: 16 where the columns make a workgroup per compute unit anyway and four
// would leave wavefronts without a piece of the reduction, if it is one turn, or a pair of filters to read (bf16, us, 4 / 16
// columns: 1024 -> 4096 3.8 / 3.3, pair 2048 -> 8192 16.0 / 12.6; 2048 -> 8192 7.8 / 8.5, 4096 -> 4096 7.6 / 8.6, 8192 -> 512 4.7 / 10.6).
bool few_columns(int f32, int gated, int M, int N, int K)
{
    const int turn = FEW_WAVES * 4 * 64 / (f32 ? 4 : 2);     // of 16 columns; of four, four times as long
    const bool filled = (N + 15) / 16 >= device_cu_count(), idle = K < 4 * turn;
    return M <= 4 && !(filled && idle && (gated || K <= turn));
}

}  // namespace

// Blocks of rows a workgroup, and the estimate in us that they are the least of, fitted to 17 .. 1500 rows of 64 x 64 to 4400 x 4368
// filters (within 10 % where it decides): 2 us, and per workgroup with 1, 2, 4 blocks the times below, once and for each turn of
// 1024 k in bf16, 512 k in fp32; what does not fit on the compute units at once takes that times `more` again (two workgroups of
// at most 128 registers share one). Fewer blocks read W more often and use more compute units: 64 rows of 2000 x 296 take
// 7.6 / 10.5 / 17.6 us in fp32 with 1 / 2 / 4 blocks, 5.0 / 6.4 / 9.4 in bf16.
// A long reduction of few workgroups is cut over workgroups, at the cost of a second launch: 8 x 8192 x 1000 fp32 25.4 -> 11.5
// us. (Only with one block of rows: with more the estimate was 1.5 times too low at 8192 k.)
struct FewBlocks {
    int blocks;      // of 16 rows a workgroup: 1, 2 or 4
    int cuts, per;   // pieces of the reduction; turns of a piece
    double us;
};
static FewBlocks few_blocks(int f32, int gated, int M, int N, int K)
{
    static constexpr double group_us[2][2][3] = {{{0.35, 0.6, 1.1}, {0.5, 1.0, 1.9}}, {{0.25, 0.5, 0.65}, {0.4, 0.9, 1.75}}};
    static constexpr double turn_us[2][2][3] = {{{1.4, 1.9, 2.65}, {2.2, 2.65, 3.2}}, {{1.45, 2.2, 4.8}, {2.5, 4.1, 7.4}}};
    static constexpr double more[2][2][3] = {{{0.7, 0.75, 0.9}, {0.85, 0.9, 1.45}}, {{0.8, 0.9, 0.9}, {0.95, 0.95, 1.2}}};
    const int t = f32 != 0, g = gated != 0;
    const long cus = device_cu_count() > 0 ? device_cu_count() : 1;
    const int length = f32 ? 512 : 1024, whole = (K + length - 1) / length;
    const double odd = !f32 && K % 2 ? 1.6 : 1.0;      // (rows one behind the other then begin in the middle of a word)
    FewBlocks best{4, 1, std::max(1, whole), 1e30};
    for (int b = M <= 16 ? 0 : 2; b >= 0; b--) {
        const long rows = (M + (16l << b) - 1) / (16l << b), groups = ((long)N + 15) / 16 * rows;
        if (rows > 65535) continue;   // (the grid's second dimension)
        for (int cuts = 1; cuts <= (b == 0 ? 8 : 1); cuts *= 2) {
            const int per = std::max(1, (whole + cuts - 1) / cuts);
            if (cuts > 1 && (groups * cuts > cus || (whole + per - 1) / per != cuts)) break;
            const double turns = cuts == 1 ? (double)K / length : per;
            const double group = group_us[t][g][b] + (turns < 0.25 ? 0.25 : turns) * turn_us[t][g][b];
            double us = 2.0 + group * odd * (1.0 + more[t][g][b] * (double)((groups * cuts + cus - 1) / cus - 1));
            if (cuts > 1) us += 2.5 + (double)cuts * M * N * (g ? 16 : 8) / 4.2e6;
            if (us < best.us) best = FewBlocks{1 << b, cuts, per, us};
        }
    }
    return best;
}
size_t dense_few_rows_piece_bytes(int f32, int gated, int M, int N, int K)
{
    if (few_columns(f32, gated, M, N, K)) return 0;
    const FewBlocks plan = few_blocks(f32, gated, M, N, K);
    return plan.cuts > 1 ? (size_t)plan.cuts * (gated ? 2 : 1) * M * ((N + 3) & ~3) * 4 : 0;
}
double dense_few_rows_us(int f32, int gated, int M, int N, int K) { return few_blocks(f32, gated, M, N, K).us; }

// Up to 16 rows always this kernel: W is the time, and it is read once and as it is. Else the least estimate. Measured, us, bf16
// through (few rows / short / tiles): 384 x 96 x 4368 19 / 6.6 / 9.2, 384 x 1000 x 64 6.0 / 12 / 8.8, 1500 x 1000 x 320 9.9 /
// 12.5 / 13.9; fp32 384 x 96 x 4368 20 / 13.8 / 16.7, 384 x 520 x 1344 12 / 17.8 / 20.9, 128 x 4096 x 4096 bf16 39 / - / 20.
DenseForm dense_forward_form(int f32, int gated, int M, int N, int K)
{
    if (M <= 16) return DENSE_FEW_ROWS;
    // (rows of bf16 that are no whole 16-byte chunks are copied for the tile kernels)
    const double copies = !f32 && K % 8 ? 6.0 + ((double)M + N) * K * 4 / 4e6 : 0.0;
    const double few = dense_few_rows_us(f32, gated, M, N, K), brief = dense_short_us(f32, gated, M, N, K);
    if (std::min(few, brief) < DENSE_LEAST_TILES_US) return few <= brief ? DENSE_FEW_ROWS : DENSE_SHORT;   // (the plan takes longer than the others)
    const double tiles = dense_product_us(M, N, K, f32, 1, gated) + copies;
    return tiles <= few && tiles <= brief ? DENSE_TILES_FORM : few <= brief ? DENSE_FEW_ROWS : DENSE_SHORT;
}

namespace {

template <typename T, bool ODD, bool GATED>
hipError_t launch_few(hipStream_t s, const DenseFewRows &given)
{
    DenseFewRows a = given;
    const bool f32 = sizeof(T) == 4;
    a.cuts = 1;
    a.per = 1 << 30;
    auto launch = [&](auto kernel, int columns, int rows) {
        const dim3 grid((unsigned)((a.N + columns - 1) / columns), (unsigned)((a.M + rows - 1) / rows), (unsigned)a.cuts);
        hipLaunchKernelGGL(kernel, grid, dim3(FEW_WAVES * 64), 0, s, a);
    };
    if (few_columns(f32, GATED, a.M, a.N, a.K)) {
        launch(dense_few_rows_kernel<T, ODD, GATED, 1, 4>, 4, 16);
        return hipGetLastError();
    }
    const FewBlocks plan = few_blocks(f32, GATED, a.M, a.N, a.K);
    if (plan.cuts > 1) {
        if (a.pieces == nullptr || a.piece_bytes < dense_few_rows_piece_bytes(f32, GATED, a.M, a.N, a.K)) return hipErrorInvalidValue;
        a.cuts = plan.cuts;
        a.per = plan.per;
    }
    if (plan.blocks == 1) launch(dense_few_rows_kernel<T, ODD, GATED, 1, 16>, 16, 16);
    else if (plan.blocks == 2) launch(dense_few_rows_kernel<T, ODD, GATED, 2, 16>, 16, 32);
    else launch(dense_few_rows_kernel<T, ODD, GATED, 4, 16>, 16, 64);
    if (a.cuts > 1) {   // (few workgroups, so few elements: their quads are counted in 31 bits)
        const long row = (a.N + 3) / 4;
        hipLaunchKernelGGL((dense_few_sum_kernel<T, GATED>), dim3((unsigned)((a.M * row + 255) / 256)), dim3(256), 0, s, a, make_fastdiv((uint32_t)row));
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_dense_few_rows(hipStream_t s, const DenseFewRows &a)
{
    if (a.M <= 0 || a.N <= 0) return hipSuccess;
    if (a.f32) return a.gated ? launch_few<float, false, true>(s, a) : launch_few<float, false, false>(s, a);
    if (odd_rows({a.X, a.W, a.W2}, {a.M > 1 ? a.ldX : 0, a.ldW, a.gated ? a.ldW2 : 0})) return a.gated ? launch_few<__bf16, true, true>(s, a) : launch_few<__bf16, true, false>(s, a);
    return a.gated ? launch_few<__bf16, false, true>(s, a) : launch_few<__bf16, false, false>(s, a);
}

}  // namespace alpha
