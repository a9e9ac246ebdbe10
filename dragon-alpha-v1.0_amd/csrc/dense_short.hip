// The dense product for short reductions or few tiles: no copy of an operand, no LDS, no barrier, one launch. What the tile
// kernels spend on filling their pipeline and on their one workgroup a compute unit is most of such a product.
//
// A workgroup of four wavefronts computes 64 x 64 of the output (a gated pair: 64 x 32 of each), each wavefront 32 x 32 (32 x 16
// of each) over the whole reduction. Both operands go straight from memory into the MFMA registers in pieces of 256 bytes of
// every row, the next piece asked for before the MFMAs of this one: bf16 v_mfma_f32_16x16x32_bf16, fp32 v_mfma_f32_16x16x4_f32,
// plain fp32 products. Neighbouring wavefronts read the same rows, from L1. A lane ends with four consecutive columns of a row.
// Rows may begin at any element and K may be any number of at least one load (16 bytes).
// Bound by the latency of a piece's loads (about 1 us bf16, 1.5 us fp32) while there is less than a workgroup a compute unit, by the
// fp32 MFMAs beyond. Measured: fp32 384 x 96 x 4368 13.8 us (16.7 through tiles), bf16 384 x 32 x 1344 5.0 (8.2).
#include "dense_direct.hpp"

namespace alpha {

template <typename T, bool ODD, bool GATED>
__global__ __launch_bounds__(256) void dense_short_kernel(const DenseFewRows a)
{
    typedef typename FewVec<T>::type vec;
    constexpr int V = 16 / sizeof(T), CHUNK = 4 * V, PIECE = 4 * CHUNK;       // k of a lane, of an MFMA's operands, of a turn
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, q = lane >> 4;
    const int m0 = blockIdx.y * 64 + (wave >> 1) * 32, n0 = GATED ? blockIdx.x * 32 + (wave & 1) * 16 : blockIdx.x * 64 + (wave & 1) * 32;
    if (m0 >= a.M || n0 >= a.N) return;
    const T *row[4];       // two blocks of rows of X, two of W or one of each filter
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int m = m0 + 16 * i + l16, n = n0 + (GATED ? 0 : 16 * i) + l16;
        row[i] = static_cast<const T *>(a.X) + (m < a.M ? m : a.M - 1) * a.ldX;
        row[2 + i] = static_cast<const T *>(GATED && i ? a.W2 : a.W) + (n < a.N ? n : a.N - 1) * (GATED && i ? a.ldW2 : a.ldW);
    }
    floatx4 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 2; j++) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};

    // (bf16, rows that begin with a word: the last load of a row ends with the word of its last element)
    const int end = sizeof(T) == 2 && !ODD ? (a.K + 1) & ~1 : a.K, last = end - V;
    auto load = [&](int k0, vec (&v)[4][4]) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const int k = k0 + c * CHUNK + q * V;
#pragma unroll
            for (int r = 0; r < 4; r++) v[c][r] = few_load<ODD>(row[r], k < last ? k : last);
        }
    };
    auto multiply = [&](int k0, vec (&v)[4][4]) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
            if (k0 + c * CHUNK >= a.K) break;
            if (k0 + (c + 1) * CHUNK > a.K) {
#pragma unroll
                for (int r = 0; r < 4; r++) v[c][r] = few_at_edge<T, ODD>(v[c][r], k0 + c * CHUNK + q * V, end, a.K);
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < 2; j++) acc[i][j] = few_multiply(v[c][2 + j], v[c][i], acc[i][j]);
        }
    };
    vec even[4][4], odd[4][4];
    load(0, even);
    for (int k0 = 0; k0 < a.K; k0 += 2 * PIECE) {
        if (k0 + PIECE < a.K) load(k0 + PIECE, odd);
        multiply(k0, even);
        if (k0 + 2 * PIECE < a.K) load(k0 + 2 * PIECE, even);
        if (k0 + PIECE < a.K) multiply(k0 + PIECE, odd);
    }

    // lane (l16, q): row l16 of a block of rows, columns 4 q .. 4 q + 3 of a block of columns
#pragma unroll 1
    for (int i = 0; i < 2; i++) {
        const int m = m0 + 16 * i + l16;
        if (m >= a.M) break;
#pragma unroll 1
        for (int j = 0; j < (GATED ? 1 : 2); j++) {
            const int n = n0 + 16 * j + 4 * q;
            if (n >= a.N) break;
            const floatx4 x = i ? (j ? acc[1][1] : acc[1][0]) : j ? acc[0][1] : acc[0][0], y = i ? acc[1][1] : acc[0][1];
            float v[4] = {x[0], x[1], x[2], x[3]}, u[4] = {y[0], y[1], y[2], y[3]};
            const bool whole = a.ep.vec && n + 4 <= a.N;
            const int left = a.N - n < 4 ? a.N - n : 4;
            if constexpr (GATED) {
                if (whole) dense_finish_gated<T, 4, true>(a.ep, v, u, m, n);
                else dense_finish_gated<T, 4, false>(a.ep, v, u, m, n, left);
            } else {
                if (whole) dense_finish<T, 4, true, true>(a.ep, v, m, n);
                else dense_finish<T, 4, true, false>(a.ep, v, m, n, left);
            }
        }
    }
}

// Estimate in us, fitted as dense_few_rows_us was: a start, the latency of a piece of the reduction (128 k of bf16, 64 of fp32), and
// from about a third of a workgroup per compute unit on what each more of them costs, by its epilogue and by its MFMAs and loads.
double dense_short_us(int f32, int gated, int M, int N, int K)
{
    if (K < (f32 ? 4 : 8) || ((long)M + 63) / 64 > 65535) return 1e30;   // (less than one load; the grid's second dimension)
    static constexpr double start[2][2] = {{3.8, 3.15}, {4.2, 3.5}}, piece[2][2] = {{0.95, 0.95}, {1.5, 1.55}};
    static constexpr double group[2][2] = {{1.4, 1.2}, {1.7, 1.3}}, by_k[2][2] = {{0.63, 0.52}, {1.75, 2.1}}, share[2][2] = {{0.3, 0.44}, {0.33, 0.72}};
    const int t = f32 != 0, g = gated != 0, cus = device_cu_count() > 0 ? device_cu_count() : 1;
    const double per_cu = (double)((N + (gated ? 31 : 63)) / (gated ? 32 : 64)) * ((M + 63) / 64) / cus - share[t][g];
    const double odd = !f32 && K % 2 ? 1.3 : 1.0;      // (as for few rows)
    const int turn = f32 ? 64 : 128;
    return odd * (start[t][g] + (double)((K + turn - 1) / turn) * piece[t][g] + (per_cu > 0 ? per_cu * (group[t][g] + K / 64.0 * by_k[t][g]) : 0.0));
}

hipError_t launch_dense_short(hipStream_t s, const DenseFewRows &a)
{
    if (a.M <= 0 || a.N <= 0) return hipSuccess;
    const dim3 grid((unsigned)((a.N + (a.gated ? 31 : 63)) / (a.gated ? 32 : 64)), (unsigned)((a.M + 63) / 64)), block(256);
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, a); };
    if (a.f32) launch(a.gated ? dense_short_kernel<float, false, true> : dense_short_kernel<float, false, false>);
    else if (odd_rows({a.X, a.W, a.W2}, {a.ldX, a.ldW, a.gated ? a.ldW2 : 0})) launch(a.gated ? dense_short_kernel<__bf16, true, true> : dense_short_kernel<__bf16, true, false>);
    else launch(a.gated ? dense_short_kernel<__bf16, false, true> : dense_short_kernel<__bf16, false, false>);
    return hipGetLastError();
}

}  // namespace alpha
