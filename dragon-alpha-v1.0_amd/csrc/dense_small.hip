// The products of a small backward: deltaX = deltaZ W and deltaW = deltaZ^T X where a tile kernel's beginning, end and second
// launch would be most of the time. Both operands straight from memory, no LDS before the end, one launch, or a second where a long
// reduction of few results is cut over workgroups.
//
// A workgroup of eight wavefronts computes 32 x 64 or 16 x 32 of C[m, n] = sum_k A(m, k) B(n, k); every wavefront takes every eighth
// chunk of k for the whole of it, and the eight sums are added through LDS in a fixed order. B has k as its rows: a lane loads
// TN columns n0 + TN (lane % 16) .. of a row, which are its elements of TN MFMAs (column TN i + j for i = lane % 16 of
// MFMA j); A with k as its rows likewise with TM columns, else a lane's consecutive k of a row. Bound by what a compute unit
// loads (35 to 40 bytes a nanosecond), in fp32 with the larger tile by the MFMAs.
//   fp32: chunks of 16 k, v_mfma_f32_16x16x4_f32, the lane's k being 4 (lane / 16) + s in the s-th: plain fp32 products;
//   bf16: chunks of 32 k, v_mfma_f32_16x16x32_bf16, eight k a lane, brought together from eight rows by byte permutes.
// Rows beyond K are zeros, rows and columns of C beyond its edge are not stored (their loads stay inside the operand).
#include "dense_finish.hpp"

#include <algorithm>

namespace alpha {

namespace {

constexpr int SMALL_WAVES = 8;

}  // namespace

struct DenseSmallArgs {
    const void *A[2], *B[2];
    long ldA, ldB;
    int M, N, K, sources;
    int per;              // chunks of a workgroup
    int cuts;             // pieces of the reduction
    int across, down;     // workgroups of a piece
    FastDiv by_row, by_piece;
    float *pieces;        // cuts > 1: [cuts][M][columns, a multiple of 4]
    DenseEpilogue ep;
};


// TM x TN: MFMA tiles of a workgroup, 2 x 4 or 1 x 2. `part`: SMALL_WAVES * TM * TN * 64 in LDS.
template <typename T, bool AT, int TM, int TN>
static __device__ __forceinline__ void small_tile(const DenseSmallArgs &a, int block, floatx4 *lds)
{
    constexpr int SMALL_M = 16 * TM, SMALL_N = 16 * TN;
    constexpr int CHUNK = sizeof(T) == 4 ? 16 : 32, V = CHUNK / 4;   // k of a chunk, of a lane
    floatx4(*const part)[TM * TN][64] = reinterpret_cast<floatx4(*)[TM * TN][64]>(lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, q = lane >> 4;
    const int piece = a.cuts > 1 ? (int)fdiv((uint32_t)block, a.by_piece) : 0, tile = block - piece * (int)a.by_piece.d;
    const int row = (int)fdiv((uint32_t)tile, a.by_row), m0 = row * SMALL_M, n0 = (tile - row * (int)a.by_row.d) * SMALL_N;
    floatx4 acc[TM][TN];
#pragma unroll
    for (int t = 0; t < TM; t++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[t][j] = floatx4{0.f, 0.f, 0.f, 0.f};

    const int chunks = (a.K + CHUNK - 1) / CHUNK;
    const bool edge_m = m0 + SMALL_M > a.M, edge_n = n0 + SMALL_N > a.N;
    const int all = chunks * a.sources, from = piece * a.per, to = from + a.per < all ? from + a.per : all;
    for (int c = from + wave; c < to; c += SMALL_WAVES) {
        const bool second = c >= chunks;
        const T *A = static_cast<const T *>(second ? a.A[1] : a.A[0]), *B = static_cast<const T *>(second ? a.B[1] : a.B[0]);
        const int k0 = (second ? c - chunks : c) * CHUNK, k = k0 + q * V;     // the chunk's first, the lane's first
        T b[V][TN], x[TM][V], xt[V][TM];                                       // x[t]: A's tile t
#pragma unroll
        for (int s = 0; s < V; s++) load_columns<TN>(B + (k + s < a.K ? k + s : a.K - 1) * a.ldB, n0 + TN * l16, a.N, b[s]);
        if constexpr (AT) {
#pragma unroll
            for (int s = 0; s < V; s++) load_columns<TM>(A + (k + s < a.K ? k + s : a.K - 1) * a.ldA, m0 + TM * l16, a.M, xt[s]);
        } else {
#pragma unroll
            for (int t = 0; t < TM; t++) {
                const int m = m0 + 16 * t + l16;
                load_columns<V>(A + (m < a.M ? m : a.M - 1) * a.ldA, k, a.K, x[t]);
            }
        }
        // edges, each uniform; what lies beyond K must be zero in both operands, columns beyond C's edge are not stored
        if (edge_n) {
#pragma unroll
            for (int s = 0; s < V; s++) at_edge<TN>(n0 + TN * l16, a.N, b[s]);
        }
        if constexpr (AT) {
            if (edge_m) {
#pragma unroll
                for (int s = 0; s < V; s++) at_edge<TM>(m0 + TM * l16, a.M, xt[s]);
            }
#pragma unroll
            for (int s = 0; s < V; s++)
#pragma unroll
                for (int t = 0; t < TM; t++) x[t][s] = xt[s][t];
        }
        if (k0 + CHUNK > a.K) {
#pragma unroll
            for (int s = 0; s < V; s++) {
                const bool there = k + s < a.K;
#pragma unroll
                for (int j = 0; j < TN; j++) b[s][j] = there ? b[s][j] : (T)0.f;
                if constexpr (AT) {
#pragma unroll
                    for (int t = 0; t < TM; t++) x[t][s] = there ? x[t][s] : (T)0.f;
                }
            }
            if constexpr (!AT) {
#pragma unroll
                for (int t = 0; t < TM; t++) at_edge<V>(k, a.K, x[t]);
            }
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int s = 0; s < V; s++)
#pragma unroll
                for (int t = 0; t < TM; t++)
#pragma unroll
                    for (int j = 0; j < TN; j++) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[s][j], x[t][s], acc[t][j], 0, 0, 0);
        } else {
            bf16x8 fx[TM];
#pragma unroll
            for (int t = 0; t < TM; t++)
#pragma unroll
                for (int s = 0; s < 8; s++) fx[t][s] = x[t][s % V];
#pragma unroll
            for (int j = 0; j < TN; j++) {
                bf16x8 fb;
#pragma unroll
                for (int s = 0; s < 8; s++) fb[s] = b[s % V][j];
#pragma unroll
                for (int t = 0; t < TM; t++) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb, fx[t], acc[t][j], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < TM; t++)
#pragma unroll
        for (int j = 0; j < TN; j++) part[wave][t * TN + j][lane] = acc[t][j];
    __syncthreads();
    // MFMA (t, j): lane (l16, q), element e: column i = 4 q + e of the MFMA, which is n0 + TN i + j; row l16, which is m0 + 16 t +
    // l16, or m0 + TM l16 + t where A has k as its rows. A thread takes TN consecutive columns of a row: one i, j = 0 .. TN - 1.
    const int part_row = threadIdx.x >> 4, i = threadIdx.x & 15;
    const int m = m0 + part_row, n = n0 + TN * i;
    if (part_row >= SMALL_M || m >= a.M || n >= a.N) return;
    const int t = AT ? part_row % TM : part_row >> 4, at = (i >> 2) * 16 + (AT ? part_row / TM : part_row & 15);
    float v[TN];
#pragma unroll
    for (int j = 0; j < TN; j++) {
        v[j] = 0.f;
#pragma unroll
        for (int w = 0; w < SMALL_WAVES; w++) v[j] += reinterpret_cast<const float *>(&part[w][t * TN + j][at])[i & 3];
    }
    if (a.cuts > 1) {
        const long columns = (a.N + 3) & ~3;
        float *to = a.pieces + ((long)piece * a.M + m) * columns + n;
#pragma unroll
        for (int j = 0; j < TN; j++)
            if (n + j < columns) to[j] = v[j];
        return;
    }
    if constexpr (TN == 4) {
        if (a.ep.vec && n + 4 <= a.N) {
            dense_finish<T, 4, false, true>(a.ep, v, m, n);
            return;
        }
    }
    dense_finish<T, TN, false, false>(a.ep, v, m, n, a.N - n < TN ? a.N - n : TN);
}

// deltaX and deltaW of one call, or one of them (the other has no workgroups): as one launch they run side by side (12 x 832 x 512
// gated bf16 backward 14.4 -> 10.7 us). BIG: tiles of 32 x 64, else 16 x 32; one launch has one size, as the larger one's LDS leaves
// room for two workgroups a compute unit only.
template <typename T, bool BIG>
__global__ __launch_bounds__(SMALL_WAVES * 64) void dense_small_kernel(const DenseSmallArgs x, const DenseSmallArgs w)
{
    constexpr int TM = BIG ? 2 : 1, TN = BIG ? 4 : 2;
    __shared__ floatx4 lds[SMALL_WAVES * TM * TN * 64];
    const int of_x = x.across * x.down * x.cuts;
    if ((int)blockIdx.x < of_x) small_tile<T, false, TM, TN>(x, blockIdx.x, lds);
    else small_tile<T, true, TM, TN>(w, blockIdx.x - of_x, lds);
}

// Adds the pieces of cut reductions in their order: four columns a thread, blocks_x workgroups for x, the others for w.
template <typename T>
static __device__ __forceinline__ void small_sum(const DenseSmallArgs &a, int block, const FastDiv &d)
{
    const long i = (long)block * 256 + threadIdx.x;
    const long m = fdiv((uint32_t)i, d), columns = (a.N + 3) & ~3;
    if (m >= a.M) return;
    const int n = (int)(i - m * d.d) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = 0; p < a.cuts; p++) {
        const floatx4 t = quad_load(a.pieces + ((long)p * a.M + m) * columns + n);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] += t[e];
    }
    if (a.ep.vec && n + 4 <= a.N) dense_finish<T, 4, false, true>(a.ep, v, m, n);
    else dense_finish<T, 4, false, false>(a.ep, v, m, n, a.N - n < 4 ? a.N - n : 4);
}
template <typename T>
__global__ __launch_bounds__(256) void dense_small_sum_kernel(const DenseSmallArgs x, const DenseSmallArgs w, int blocks_x, FastDiv d_x, FastDiv d_w)
{
    if ((int)blockIdx.x < blocks_x) small_sum<T>(x, blockIdx.x, d_x);
    else small_sum<T>(w, blockIdx.x - blocks_x, d_w);
}

namespace {

// Tile and cut of the reduction with the least estimate, which is in us.
struct SmallPlan {
    bool few;        // the smaller tile
    int pieces, per; // per: chunks
    double us;
};
// Estimate, fitted to products of 16 .. 4400 x 32 .. 3000 x 32 .. 4400 (within 10 % in fp32, 20 % in bf16): a start, the reduction by
// k (fp32: 4 / 7 ns with the smaller and larger tile) or turns of 128 (bf16: 0.33 / 0.57 us), and as much as that again and an
// epilogue for every workgroup a compute unit; a cut costs a second launch and the pieces' way through memory. Measured, smaller
// / larger / tile kernels: 200 x 240 x 760 bf16 4.1 / 6.0 / 10.0, fp32 5.8 / 11.6 / 12.5; 200 x 3000 x 1500 deltaW bf16 38 / 21 /
// 17; 64 x 320 of two reductions of 3136 fp32, in one piece and cut: 36.5 / 14.5.
SmallPlan small_plan(int f32, int M, int N, int K, int sources)
{
    const long cus = device_cu_count() > 0 ? device_cu_count() : 1;
    const int size = f32 ? 16 : 32, chunks = (K + size - 1) / size * sources;
    SmallPlan best{false, 1, std::max(1, chunks), 1e30};
    for (int few = 0; few < 2; few++) {
        const long groups = few ? ((long)M + 15) / 16 * ((N + 31) / 32) : ((long)M + 31) / 32 * ((N + 63) / 64);
        for (int pieces = 1; pieces <= 16; pieces *= 2) {
            // (every piece of at least two turns of the eight wavefronts)
            const int per = (chunks + pieces - 1) / pieces;
            if (pieces > 1 && (groups * pieces > cus || per < 16 || (chunks + per - 1) / per != pieces)) break;
            const double length = f32 ? per * 16.0 : (double)((per + 3) / 4), per_cu = (double)groups * pieces / cus;
            double us = f32 ? (few ? 2.25 + length * 0.004 + per_cu * (0.23 + length * 0.004) : 3.05 + length * 0.007 + per_cu * (1.2 + length * 0.011))
                            : (few ? 2.2 + length * 0.33 + per_cu * (0.06 + length * 0.37) : 2.8 + length * 0.57 + per_cu * (1.4 + length * 0.35));
            if (pieces > 1) us += 2.5 + (double)pieces * M * N * 8 / 4.2e6;
            if (us < best.us) best = SmallPlan{few != 0, pieces, per, us};
        }
    }
    return best;
}

}  // namespace

size_t dense_small_piece_bytes(int f32, int M, int N, int K, int sources)
{
    const SmallPlan plan = small_plan(f32, M, N, K, sources);
    return plan.pieces > 1 ? (size_t)plan.pieces * M * ((N + 3) & ~3) * 4 : 0;
}

// By the estimates. (A load at an edge takes what lies before it, so rows have at least one load: of columns of B, and of columns or
// k of A.)
bool dense_small_preferred(int f32, int a_t, int M, int N, int K, int sources)
{
    // (rows of bf16 that are no whole 16-byte chunks are copied for the tile kernels)
    const double copies = !f32 && N % 8 ? 3.0 + (double)K * sources * N * 4 / 4e6 : 0.0;
    if (N < 4 || K < 1 || (a_t ? M < 2 : K < 8) || ((long)M + 15) / 16 > 65535) return false;   // (65535: the grid's second dimension)
    const double us = small_plan(f32, M, N, K, sources).us;
    return us < DENSE_LEAST_TILES_US || us < dense_product_us(M, N, K, f32, sources, 0) + copies;
}

namespace {

// One product's arguments; pieces: room for them, taken from its beginning. big: its tile.
DenseSmallArgs small_args(const DenseProduct &p, float *&pieces, bool &big)
{
    const SmallPlan plan = small_plan(p.f32, p.M, p.N, p.K, p.sources);
    DenseSmallArgs a{};
    for (int i = 0; i < 2; i++) {
        a.A[i] = p.A.p[i];
        a.B[i] = p.B.p[i];
    }
    a.ldA = p.A.ld;
    a.ldB = p.B.ld;
    a.M = p.M;
    a.N = p.N;
    a.K = p.K;
    a.sources = p.sources;
    a.ep = p.ep;
    a.per = plan.per;
    a.cuts = plan.pieces;
    big = !plan.few;
    a.across = (p.N + (big ? 63 : 31)) / (big ? 64 : 32);
    a.down = (p.M + (big ? 31 : 15)) / (big ? 32 : 16);
    a.by_row = make_fastdiv((uint32_t)a.across);
    a.by_piece = make_fastdiv((uint32_t)std::min<long>((long)a.across * a.down, (1l << 31) - 1));
    a.pieces = pieces;
    if (plan.pieces > 1) pieces += (long)plan.pieces * p.M * ((p.N + 3) & ~3);
    return a;
}

}  // namespace

// x: A straight; w: A with k as its rows; either may be null, but not both.
hipError_t launch_dense_small(hipStream_t s, const DenseProduct *px, const DenseProduct *pw)
{
    const DenseProduct &any = px ? *px : *pw;
    float *pieces = any.pieces;
    size_t need = 0;
    for (const DenseProduct *p : {px, pw})
        if (p) need += dense_small_piece_bytes(p->f32, p->M, p->N, p->K, p->sources);
    if (need > 0 && (pieces == nullptr || any.piece_bytes < need)) return hipErrorInvalidValue;
    bool big_x = false, big_w = false;
    const DenseSmallArgs x = px ? small_args(*px, pieces, big_x) : DenseSmallArgs{}, w = pw ? small_args(*pw, pieces, big_w) : DenseSmallArgs{};
    hipError_t e = hipSuccess;
    auto run = [&](bool big, const DenseSmallArgs &x, const DenseSmallArgs &w) {
        const long blocks = (long)x.across * x.down * x.cuts + (long)w.across * w.down * w.cuts;
        if (blocks >= (1l << 31)) e = hipErrorInvalidValue;
        if (e != hipSuccess) return;
        auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(SMALL_WAVES * 64), 0, s, x, w); };
        if (any.f32) launch(big ? dense_small_kernel<float, true> : dense_small_kernel<float, false>);
        else launch(big ? dense_small_kernel<__bf16, true> : dense_small_kernel<__bf16, false>);
    };
    if (px && pw && big_x != big_w) {
        run(big_x, x, DenseSmallArgs{});
        run(big_w, DenseSmallArgs{}, w);
    } else {
        run(px ? big_x : big_w, x, w);
    }
    if (e != hipSuccess) return e;
    if (need > 0) {   // (few workgroups, so few elements: their quads are counted in 31 bits)
        auto sums = [](const DenseSmallArgs &a) { return a.cuts > 1 ? (unsigned)(((long)a.M * ((a.N + 3) / 4) + 255) / 256) : 0u; };
        const unsigned of_x = sums(x), of_w = sums(w);
        const FastDiv d_x = make_fastdiv((uint32_t)std::max(1, (x.N + 3) / 4)), d_w = make_fastdiv((uint32_t)std::max(1, (w.N + 3) / 4));
        if (any.f32) hipLaunchKernelGGL((dense_small_sum_kernel<float>), dim3(of_x + of_w), dim3(256), 0, s, x, w, (int)of_x, d_x, d_w);
        else hipLaunchKernelGGL((dense_small_sum_kernel<__bf16>), dim3(of_x + of_w), dim3(256), 0, s, x, w, (int)of_x, d_x, d_w);
    }
    return hipGetLastError();
}

}  // namespace alpha
