// The dense product for few rows of X or little work: no copy of an operand, one launch, as many bytes in flight as the
// device takes. A single row reads W once and is bound by that.
//
// A workgroup of eight wavefronts computes 16 columns of the output (16 rows of W) for up to 64 rows of X; its wavefronts
// share the reduction in pieces of 256 bytes of every row. Both operands go straight from memory into the MFMA registers: a
// lane holds 16 bytes of one row of W and of one row of X at the same k. bf16: v_mfma_f32_16x16x32_bf16, eight k a lane;
// fp32: v_mfma_f32_16x16x4_f32, component s of the lane's four k in the s-th MFMA - plain fp32 products. Rows of X beyond
// the last are the last once more, their results not stored. The partial sums are added through LDS in a fixed order.
// At most four rows of X: four columns a workgroup instead of 16, the MFMA's 16 rows and columns being four pieces of the
// reduction times four (only the products of equal pieces are read out): four times as many workgroups, each with a
// quarter of the reduction's length in turns (1 x 8192 x 1024 of bf16: 11.4 -> 5.4 us).
// Rows may begin at any element and K may be any number.
#include "dense_finish.hpp"

namespace alpha {

namespace {

constexpr int FEW_WAVES = 8;

template <typename T> struct FewVec;
template <> struct FewVec<float> { typedef floatx4 type; };
template <> struct FewVec<__bf16> { typedef bf16x8 type; };

// 16 bytes of a row from element k on, whatever its alignment
template <typename T>
__device__ __forceinline__ typename FewVec<T>::type few_load(const T *row, int k)
{
    typename FewVec<T>::type v;
    __builtin_memcpy(&v, row + k, 16);
    return v;
}
// what was loaded at K - V instead of at k > K - V, moved to its place: zeros from K on
template <typename T>
__device__ __forceinline__ typename FewVec<T>::type few_at_edge(typename FewVec<T>::type x, int k, int K)
{
    constexpr int V = 16 / sizeof(T);
    T v[V];
#pragma unroll
    for (int e = 0; e < V; e++) v[e] = x[e];
    at_edge<V>(k, K, v);
#pragma unroll
    for (int e = 0; e < V; e++) x[e] = v[e];
    return x;
}

__device__ __forceinline__ floatx4 few_multiply(bf16x8 w, bf16x8 x, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x, c, 0, 0, 0); }
__device__ __forceinline__ floatx4 few_multiply(floatx4 w, floatx4 x, floatx4 c)
{
#pragma unroll
    for (int s = 0; s < 4; s++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(w[s], x[s], c, 0, 0, 0);
    return c;
}

}  // namespace

// C: columns of a workgroup, 16, or 4 for at most four rows. MB: blocks of 16 rows.
template <typename T, bool GATED, int MB, int C>
__global__ __launch_bounds__(FEW_WAVES * 64) void dense_few_rows_kernel(const DenseFewRows a)
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
    const int turns = a.K < V ? 0 : (a.K + FEW_WAVES * SPAN - 1) / (FEW_WAVES * SPAN);
    int turn = turns > 0 ? (int)(blockIdx.x % turns) : 0;
    for (int t = 0; t < turns; t++) {
        const int k0 = (turn * FEW_WAVES + wave) * SPAN, k = k0 + l16 / C * PIECE;
        if (k0 < a.K) {
            vec vw[G][4], vx[MB][4];
            const int last = a.K - V;      // >= 0
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int at = k + c * CHUNK + q * V;
#pragma unroll
                for (int g = 0; g < G; g++) vw[g][c] = few_load(w[g], at < last ? at : last);
            }
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int at = k + c * CHUNK + q * V;
#pragma unroll
                for (int b = 0; b < MB; b++) vx[b][c] = few_load(x[b], at < last ? at : last);
            }
            const bool edge = k0 + SPAN > a.K;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                if (edge) {
#pragma unroll
                    for (int g = 0; g < G; g++) vw[g][c] = few_at_edge<T>(vw[g][c], k + c * CHUNK + q * V, a.K);
#pragma unroll
                    for (int b = 0; b < MB; b++) vx[b][c] = few_at_edge<T>(vx[b][c], k + c * CHUNK + q * V, a.K);
                }
#pragma unroll
                for (int g = 0; g < G; g++)
#pragma unroll
                    for (int b = 0; b < MB; b++) acc[g][b] = few_multiply(vw[g][c], vx[b][c], acc[g][b]);
            }
        }
        turn = turn + 1 == turns ? 0 : turn + 1;
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
        if constexpr (GATED) dense_finish_gated<T, 1, false>(a.ep, v, u, m, n0 + col);
        else dense_finish<T, 1, true, false>(a.ep, v, m, n0 + col);
    }
}

namespace {

// Four columns a workgroup or 16, for at most four rows: 16 where the columns make a workgroup per compute unit anyway and four
// would leave wavefronts without a piece of the reduction, if it is one turn, or a pair of filters to read (bf16, us, 4 / 16
// columns: 1024 -> 4096 3.8 / 3.3, pair 2048 -> 8192 16.0 / 12.6; 2048 -> 8192 7.8 / 8.5, 4096 -> 4096 7.6 / 8.6, 8192 -> 512 4.7 / 10.6).
template <typename T>
bool few_columns(const DenseFewRows &a)
{
    constexpr int TURN = FEW_WAVES * 4 * 64 / sizeof(T);     // of 16 columns; of four, four times as long
    const bool filled = (a.N + 15) / 16 >= device_cu_count(), idle = a.K < 4 * TURN;
    return !(filled && idle && (a.gated || a.K <= TURN));
}

template <typename T, bool GATED>
hipError_t launch_few(hipStream_t s, const DenseFewRows &a)
{
    const dim3 block(FEW_WAVES * 64), grid((unsigned)((a.N + 15) / 16), (unsigned)((a.M + 63) / 64));
    if (a.M <= 4 && few_columns<T>(a)) hipLaunchKernelGGL((dense_few_rows_kernel<T, GATED, 1, 4>), dim3((unsigned)((a.N + 3) / 4)), block, 0, s, a);
    else if (a.M <= 16) hipLaunchKernelGGL((dense_few_rows_kernel<T, GATED, 1, 16>), grid, block, 0, s, a);
    else if (a.M <= 32) hipLaunchKernelGGL((dense_few_rows_kernel<T, GATED, 2, 16>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((dense_few_rows_kernel<T, GATED, 4, 16>), grid, block, 0, s, a);
    return hipGetLastError();
}

}  // namespace

// Up to 16 rows always: W is the time, and this kernel reads it once and as it is. More rows: by an estimate against the tile
// kernel's. A workgroup's turn (1024 k of bf16, 512 of fp32) of 2 / 4 blocks of rows takes 2.7 / 4.7 us in bf16, 2.7 / 6.5 in
// fp32, 1.4 and 1.6 times that for a gated pair (measured on 512 x 1000 to 4096 x 4096 filters). E.g. 200 rows of 512 x 1000
// bf16: 5.4 us here, 9 to 18 through tiles; 128 rows of 4096 x 4096: 39 against 20.
bool dense_few_rows_preferred(int f32, int gated, int M, int N, int K)
{
    if (M <= 16) return true;
    if ((M + 63) / 64 > 65535) return false;   // (the grid's second dimension)
    static constexpr double turn_us[2][2] = {{2.7, 4.7}, {2.7, 6.5}};
    const int cus = device_cu_count() > 0 ? device_cu_count() : 1;
    const double groups = (double)((N + 15) / 16) * ((M + 63) / 64), turns = (double)K / (f32 ? 512 : 1024);
    const double turn = turn_us[f32 ? 1 : 0][M > 32] * (!gated ? 1.0 : f32 ? 1.6 : 1.4);
    const double us = 2.0 + (groups > cus ? groups / cus : 1.0) * (0.7 + (turns < 0.5 ? 0.5 : turns) * turn);
    return us < dense_product_us(M, N, K, f32, 1, gated);
}

hipError_t launch_dense_few_rows(hipStream_t s, const DenseFewRows &a)
{
    if (a.M <= 0 || a.N <= 0) return hipSuccess;
    if (a.gated) return a.f32 ? launch_few<float, true>(s, a) : launch_few<__bf16, true>(s, a);
    return a.f32 ? launch_few<float, false>(s, a) : launch_few<__bf16, false>(s, a);
}

}  // namespace alpha
