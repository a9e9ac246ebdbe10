// The products of a small backward: deltaX = deltaZ W and deltaW = deltaZ^T X where a tile kernel's beginning, end and second
// launch would be most of the time. Both operands straight from memory, no LDS before the end, one launch.
//
// A workgroup of eight wavefronts computes 32 x 64 of C[m, n] = sum_k A(m, k) B(n, k); every wavefront takes every eighth
// chunk of k for the whole of it, and the eight sums are added through LDS in a fixed order. B has k as its rows: a lane loads
// four columns n0 + 4 (lane % 16) .. + 3 of a row, which are its elements of four MFMAs (column 4 i + j for i = lane % 16 of
// MFMA j); A with k as its rows likewise with two columns, else a lane's consecutive k of a row.
//   fp32: chunks of 16 k, v_mfma_f32_16x16x4_f32, the lane's k being 4 (lane / 16) + s in the s-th: plain fp32 products;
//   bf16: chunks of 32 k, v_mfma_f32_16x16x32_bf16, eight k a lane, brought together from eight rows by byte permutes.
// Rows beyond K are zeros, rows and columns of C beyond its edge are not stored (their loads stay inside the operand).
#include "dense_finish.hpp"

namespace alpha {

namespace {

constexpr int SMALL_WAVES = 8;

}  // namespace

struct DenseSmallArgs {
    const void *A[2], *B[2];
    long ldA, ldB;
    int M, N, K, sources;
    DenseEpilogue ep;
};

// TM x TN: MFMA tiles of a workgroup, 2 x 4 or 1 x 2
template <typename T, bool AT, int TM, int TN>
__global__ __launch_bounds__(SMALL_WAVES * 64) void dense_small_kernel(const DenseSmallArgs a)
{
    constexpr int SMALL_M = 16 * TM, SMALL_N = 16 * TN;
    constexpr int CHUNK = sizeof(T) == 4 ? 16 : 32, V = CHUNK / 4;   // k of a chunk, of a lane
    __shared__ floatx4 part[SMALL_WAVES][TM * TN][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, q = lane >> 4;
    const int m0 = blockIdx.y * SMALL_M, n0 = blockIdx.x * SMALL_N;
    floatx4 acc[TM][TN];
#pragma unroll
    for (int t = 0; t < TM; t++)
#pragma unroll
        for (int j = 0; j < TN; j++) acc[t][j] = floatx4{0.f, 0.f, 0.f, 0.f};

    const int chunks = (a.K + CHUNK - 1) / CHUNK;
    const bool edge_m = m0 + SMALL_M > a.M, edge_n = n0 + SMALL_N > a.N;
    for (int c = wave; c < chunks * a.sources; c += SMALL_WAVES) {
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
    const int row = threadIdx.x >> 4, i = threadIdx.x & 15;
    const int m = m0 + row, n = n0 + TN * i;
    if (row >= SMALL_M || m >= a.M || n >= a.N) return;
    const int t = AT ? row % TM : row >> 4, at = (i >> 2) * 16 + (AT ? row / TM : row & 15);
    float v[TN];
#pragma unroll
    for (int j = 0; j < TN; j++) {
        v[j] = 0.f;
#pragma unroll
        for (int w = 0; w < SMALL_WAVES; w++) v[j] += reinterpret_cast<const float *>(&part[w][t * TN + j][at])[i & 3];
    }
    if constexpr (TN == 4) {
        if (a.ep.vec && n + 4 <= a.N) {
            dense_finish<T, 4, false, true>(a.ep, v, m, n);
            return;
        }
    }
    dense_finish<T, TN, false, false>(a.ep, v, m, n, a.N - n < TN ? a.N - n : TN);
}

namespace {

// The smaller tile where it is faster by the estimate, which is returned.
struct SmallTiles {
    bool few;
    double us;
};
// Estimate in us, fitted to products of 16 .. 4400 x 32 .. 3000 x 32 .. 4400 (within 10 % in fp32, 20 % in bf16): a start, the
// reduction by k (fp32: 4 / 7 ns with the smaller and larger tile) or turns of 128 (bf16: 0.33 / 0.57 us), and as much as that
// again and an epilogue for every workgroup a compute unit. Measured, smaller / larger / tile kernels: 200 x 240 x 760 bf16 4.1 /
// 6.0 / 10.0, fp32 5.9 / 11.6 / 14.1; 200 x 3000 x 1500 deltaW bf16 38 / 21 / 17.
SmallTiles small_tiles(int f32, int M, int N, int K, int sources)
{
    const long cus = device_cu_count() > 0 ? device_cu_count() : 1, all = (long)K * sources;
    const double length = f32 ? (double)all : (double)((all + 127) / 128);
    auto per_cu = [&](int m, int n) { return (double)(((long)M + m - 1) / m * ((N + n - 1) / n)) / cus; };
    const double few = f32 ? 2.25 + length * 0.004 + per_cu(16, 32) * (0.23 + length * 0.004) : 2.2 + length * 0.33 + per_cu(16, 32) * (0.06 + length * 0.37);
    const double many = f32 ? 3.05 + length * 0.007 + per_cu(32, 64) * (1.2 + length * 0.011) : 2.8 + length * 0.57 + per_cu(32, 64) * (1.4 + length * 0.35);
    return few < many ? SmallTiles{true, few} : SmallTiles{false, many};
}

}  // namespace

// By the estimates. (A load at an edge takes what lies before it, so rows have at least one load: of columns of B, and of columns or
// k of A.)
bool dense_small_preferred(int f32, int a_t, int M, int N, int K, int sources)
{
    // (rows of bf16 that are no whole 16-byte chunks are copied for the tile kernels)
    const double copies = !f32 && N % 8 ? 3.0 + (double)K * sources * N * 4 / 4e6 : 0.0;
    if (N < 4 || K < 1 || (a_t ? M < 2 : K < 8) || (M + 15) / 16 > 65535) return false;   // (65535: the grid's second dimension)
    return small_tiles(f32, M, N, K, sources).us < dense_product_us(M, N, K, f32, sources, 0) + copies;
}

hipError_t launch_dense_small(hipStream_t s, const DenseProduct &p)
{
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
    auto launch = [&](auto kernel, int tm, int tn) {
        const dim3 grid((unsigned)((p.N + 16 * tn - 1) / (16 * tn)), (unsigned)((p.M + 16 * tm - 1) / (16 * tm)));
        hipLaunchKernelGGL(kernel, grid, dim3(SMALL_WAVES * 64), 0, s, a);
    };
    if (small_tiles(p.f32, p.M, p.N, p.K, p.sources).few) {
        if (p.a_t) launch(p.f32 ? dense_small_kernel<float, true, 1, 2> : dense_small_kernel<__bf16, true, 1, 2>, 1, 2);
        else launch(p.f32 ? dense_small_kernel<float, false, 1, 2> : dense_small_kernel<__bf16, false, 1, 2>, 1, 2);
    } else {
        if (p.a_t) launch(p.f32 ? dense_small_kernel<float, true, 2, 4> : dense_small_kernel<__bf16, true, 2, 4>, 2, 4);
        else launch(p.f32 ? dense_small_kernel<float, false, 2, 4> : dense_small_kernel<__bf16, false, 2, 4>, 2, 4);
    }
    return hipGetLastError();
}

}  // namespace alpha
