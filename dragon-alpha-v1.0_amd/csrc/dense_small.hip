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

constexpr int SMALL_WAVES = 8, SMALL_M = 32, SMALL_N = 64;

}  // namespace

struct DenseSmallArgs {
    const void *A[2], *B[2];
    long ldA, ldB;
    int M, N, K, sources;
    DenseEpilogue ep;
};

template <typename T, bool AT>
__global__ __launch_bounds__(SMALL_WAVES * 64) void dense_small_kernel(const DenseSmallArgs a)
{
    constexpr int CHUNK = sizeof(T) == 4 ? 16 : 32, V = CHUNK / 4;   // k of a chunk, of a lane
    __shared__ floatx4 part[SMALL_WAVES][8][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, q = lane >> 4;
    const int m0 = blockIdx.y * SMALL_M, n0 = blockIdx.x * SMALL_N;
    floatx4 acc[2][4];
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[t][j] = floatx4{0.f, 0.f, 0.f, 0.f};

    const int chunks = (a.K + CHUNK - 1) / CHUNK;
    const bool edge_m = m0 + SMALL_M > a.M, edge_n = n0 + SMALL_N > a.N;
    for (int c = wave; c < chunks * a.sources; c += SMALL_WAVES) {
        const bool second = c >= chunks;
        const T *A = static_cast<const T *>(second ? a.A[1] : a.A[0]), *B = static_cast<const T *>(second ? a.B[1] : a.B[0]);
        const int k0 = (second ? c - chunks : c) * CHUNK, k = k0 + q * V;     // the chunk's first, the lane's first
        T b[V][4], x[2][V], xt[V][2];                                         // x[t]: A's tile t
#pragma unroll
        for (int s = 0; s < V; s++) load_columns<4>(B + (k + s < a.K ? k + s : a.K - 1) * a.ldB, n0 + 4 * l16, a.N, b[s]);
        if constexpr (AT) {
#pragma unroll
            for (int s = 0; s < V; s++) load_columns<2>(A + (k + s < a.K ? k + s : a.K - 1) * a.ldA, m0 + 2 * l16, a.M, xt[s]);
        } else {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int m = m0 + 16 * t + l16;
                load_columns<V>(A + (m < a.M ? m : a.M - 1) * a.ldA, k, a.K, x[t]);
            }
        }
        // edges, each uniform; what lies beyond K must be zero in both operands, columns beyond C's edge are not stored
        if (edge_n) {
#pragma unroll
            for (int s = 0; s < V; s++) at_edge<4>(n0 + 4 * l16, a.N, b[s]);
        }
        if constexpr (AT) {
            if (edge_m) {
#pragma unroll
                for (int s = 0; s < V; s++) at_edge<2>(m0 + 2 * l16, a.M, xt[s]);
            }
#pragma unroll
            for (int s = 0; s < V; s++) {
                x[0][s] = xt[s][0];
                x[1][s] = xt[s][1];
            }
        }
        if (k0 + CHUNK > a.K) {
#pragma unroll
            for (int s = 0; s < V; s++) {
                const bool there = k + s < a.K;
#pragma unroll
                for (int j = 0; j < 4; j++) b[s][j] = there ? b[s][j] : (T)0.f;
                if constexpr (AT) {
                    x[0][s] = there ? x[0][s] : (T)0.f;
                    x[1][s] = there ? x[1][s] : (T)0.f;
                }
            }
            if constexpr (!AT) {
                at_edge<V>(k, a.K, x[0]);
                at_edge<V>(k, a.K, x[1]);
            }
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int s = 0; s < V; s++)
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[s][j], x[t][s], acc[t][j], 0, 0, 0);
        } else {
            bf16x8 fx[2];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int s = 0; s < 8; s++) fx[t][s] = x[t][s % V];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                bf16x8 fb;
#pragma unroll
                for (int s = 0; s < 8; s++) fb[s] = b[s % V][j];
#pragma unroll
                for (int t = 0; t < 2; t++) acc[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb, fx[t], acc[t][j], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int j = 0; j < 4; j++) part[wave][t * 4 + j][lane] = acc[t][j];
    __syncthreads();
    // MFMA (t, j): lane (l16, q), element e: column i = 4 q + e of the MFMA, which is n0 + 4 i + j; row l16, which is m0 + 16 t +
    // l16, or m0 + 2 l16 + t where A has k as its rows. A thread takes four consecutive columns of a row: one i, j = 0 .. 3.
    const int row = threadIdx.x >> 4, i = threadIdx.x & 15;
    const int m = m0 + row, n = n0 + 4 * i;
    if (m >= a.M || n >= a.N) return;
    const int t = AT ? row & 1 : row >> 4, at = (i >> 2) * 16 + (AT ? row >> 1 : row & 15);
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        v[j] = 0.f;
#pragma unroll
        for (int w = 0; w < SMALL_WAVES; w++) v[j] += reinterpret_cast<const float *>(&part[w][t * 4 + j][at])[i & 3];
    }
    if (a.ep.vec && n + 4 <= a.N) {
        dense_finish<T, 4, false, true>(a.ep, v, m, n);
    } else {
        dense_finish<T, 4, false, false>(a.ep, v, m, n, a.N - n < 4 ? a.N - n : 4);
    }
}

// By an estimate against the tile kernels': a workgroup's reduction takes 12.5 ns a k in fp32 (its MFMAs), 0.9 us a turn of 256 k
// in bf16 (the loads). 100 x 2000 x 500 backward in fp32 / bf16: 14 + 14 / 13 + 8 us through tiles, 10 + 8 / 7 + 5 here.
bool dense_small_preferred(int f32, int M, int N, int K, int sources)
{
    const int cus = device_cu_count() > 0 ? device_cu_count() : 1;
    const long groups = ((long)M + SMALL_M - 1) / SMALL_M * ((N + SMALL_N - 1) / SMALL_N), rounds = (groups + cus - 1) / cus;
    const double all = (double)K * sources, us = 3.0 + rounds * (1.0 + (f32 ? all * 0.0125 : (double)(long)((all + 255) / 256) * 0.9));
    // (the loads at an edge take what lies before it)
    // (rows of bf16 that are no whole 16-byte chunks are copied for the tile kernels)
    const double copies = !f32 && N % 8 ? 3.0 + all * N * 4 / 4e6 : 0.0;
    return M >= 2 && N >= 4 && K >= 8 && (M + SMALL_M - 1) / SMALL_M <= 65535 && us < dense_product_us(M, N, K, f32, sources, 0) + copies;
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
    const dim3 grid((unsigned)((p.N + SMALL_N - 1) / SMALL_N), (unsigned)((p.M + SMALL_M - 1) / SMALL_M)), block(SMALL_WAVES * 64);
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, a); };
    if (p.a_t) launch(p.f32 ? dense_small_kernel<float, true> : dense_small_kernel<__bf16, true>);
    else launch(p.f32 ? dense_small_kernel<float, false> : dense_small_kernel<__bf16, false>);
    return hipGetLastError();
}

}  // namespace alpha
