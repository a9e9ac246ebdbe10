// Launch of the dense product: tile shape and cut of the reduction by size, the second kernel that adds the pieces.
#include "dense_gemm_launch.hpp"

#include <algorithm>

namespace alpha {

// Adds the pieces of a cut reduction in their order and applies the epilogue; one thread per four columns.
template <typename T, bool GATED>
__global__ __launch_bounds__(256) void dense_pieces_kernel(const DenseTileArgs a, long a_row, long a_k, long b_row, long b_k, FastDiv d_quads)
{
    const long quads = d_quads.d;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < quads * a.M; i += (long)gridDim.x * 256) {
        const int m = quads * a.M < (1l << 31) ? (int)fdiv((uint32_t)i, d_quads) : (int)(i / quads);
        const int n = (int)(i - m * quads) * 4;
        floatx4 v{0.f, 0.f, 0.f, 0.f}, u = v;
        const float *src = a.partial + (long)m * a.columns + n;
        for (int p = 0; p < a.split; p++, src += (long)a.M * a.columns) {
            if ((a.columns & 3) == 0 && (a.N & 3) == 0) {
                v += *reinterpret_cast<const floatx4 *>(src);
                if (GATED) u += *reinterpret_cast<const floatx4 *>(src + a.N);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (n + e < a.N) {
                        v[e] += src[e];
                        if (GATED) u[e] += src[a.N + e];
                    }
            }
        }
        if constexpr (__is_same(T, float)) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (n + e >= a.N) break;
                if (v[e] != v[e])
                    v[e] = dense_element(a.A[0], a.A[1], m * a_row, a_k, a.planeA, a.B[0], a.B[1], (n + e) * b_row, b_k, a.planeB,
                                         GATED ? 1 : a.combos / a.parts6, a.K);
                if (GATED && u[e] != u[e])
                    u[e] = dense_element(a.A[0], a.A[1], m * a_row, a_k, a.planeA, a.B[1], a.B[1], (n + e) * b_row, b_k, a.planeB, 1, a.K);
            }
        }
        float x[4] = {v[0], v[1], v[2], v[3]}, y[4] = {u[0], u[1], u[2], u[3]};
        if constexpr (GATED) dense_finish_gated<T>(a.ep, x, y, m, n, a.N);
        else dense_finish<T>(a.ep, x, m, n, a.N);
    }
}

namespace {

struct Plan {
    bool big;
    int split, per, tiles_m, tiles_n, steps;
};

// Tile shape and cut: the least of a simple estimate of the device's time. `room`: bytes for the pieces.
Plan make_plan(int M, int N, int K, int parts, int sources, int gated, size_t room)
{
    const int cus = std::max(1, device_cu_count());
    const int nk = std::max(1, (K + 31) / 32), steps = nk * (parts == 3 ? 6 : 1) * sources;
    const double out_bytes = (double)M * N * (gated ? 2 : 1) * 4;
    Plan best{};
    double best_us = 1e30;
    for (int big = 0; big < 2; big++) {
        const int bm = big ? 256 : 128, bn = (big ? 256 : 128) / (gated ? 2 : 1);
        const int tm = (M + bm - 1) / bm, tn = (N + bn - 1) / bn;
        const long tiles = (long)tm * tn, slots = (long)cus * (big ? 1 : 2);
        for (int split = 1; split <= 64; split++) {
            // whole k steps: a piece holds all parts of its products, so none leaves fp32's range that the sum would not
            // (and an even number of steps: the kernel's loop does two at a time)
            const int combos = steps / nk, per = (nk + 2 * split - 1) / (2 * split) * 2 * combos;
            if (split > 1 && (per < 8 || (long)split * M * N * (gated ? 2 : 1) * 4 > (long)room)) break;
            if ((steps + per - 1) / per != split) continue;   // every piece has a step
            const long rounds = (tiles * split + slots - 1) / slots;
            double us = rounds * (per * (big ? 0.65 : 0.4) + 3.0);
            if (split > 1) us += 3.0 + out_bytes * (split * 2 + 1) / 4e6;
            if (us < best_us) {
                best_us = us;
                best = Plan{big != 0, split, per, tm, tn, steps};
            }
        }
    }
    return best;
}

}  // namespace

size_t dense_product_partial_bytes(int M, int N, int K, int parts, int sources, int gated)
{
    // as many pieces as the plan without a limit takes
    const Plan p = make_plan(M, N, K, parts, sources, gated, (size_t)1 << 60);
    return p.split > 1 ? (size_t)p.split * M * N * (gated ? 2 : 1) * 4 : 0;
}

hipError_t launch_dense_product(hipStream_t s, const DenseProduct &p)
{
    if (p.M <= 0 || p.N <= 0) return hipSuccess;
    const Plan plan = make_plan(p.M, p.N, p.K, p.parts, p.sources, p.gated, p.partial ? p.partial_bytes : 0);
    DenseTileArgs a{};
    for (int i = 0; i < 2; i++) {
        a.A[i] = p.A.p[i];
        a.B[i] = p.B.p[i];
    }
    a.ldA = p.A.ld;
    a.ldB = p.B.ld;
    a.planeA = p.A.plane;
    a.planeB = p.B.plane;
    a.M = p.M;
    a.N = p.N;
    a.K = p.K;
    a.parts6 = p.parts == 3 ? 6 : 1;
    a.combos = a.parts6 * p.sources;
    a.steps = plan.steps;
    a.split = plan.split;
    a.per = plan.per;
    a.tiles_m = plan.tiles_m;
    a.tiles_n = plan.tiles_n;
    a.ep = p.ep;
    a.partial = p.partial;
    a.columns = p.gated ? 2 * p.N : p.N;
    hipError_t e;
    if (p.a_t) e = launch_dense_tile_tt(s, a, plan.big, p.f32);
    else if (p.b_t) e = launch_dense_tile_st(s, a, plan.big, p.f32);
    else if (p.gated) e = launch_dense_tile_gated(s, a, plan.big, p.f32);
    else e = launch_dense_tile_ss(s, a, plan.big, p.f32);
    if (e != hipSuccess || a.split == 1) return e;
    const long quads = (p.N + 3) / 4, work = quads * p.M;
    const FastDiv d = make_fastdiv((uint32_t)quads);
    const dim3 grid((unsigned)std::min<long>((work + 255) / 256, 8192));
    const long a_row = p.a_t ? 1 : p.A.ld, a_k = p.a_t ? p.A.ld : 1, b_row = p.b_t ? 1 : p.B.ld, b_k = p.b_t ? p.B.ld : 1;
    if (p.gated) {
        if (p.f32) hipLaunchKernelGGL((dense_pieces_kernel<float, true>), grid, dim3(256), 0, s, a, a_row, a_k, b_row, b_k, d);
        else hipLaunchKernelGGL((dense_pieces_kernel<__bf16, true>), grid, dim3(256), 0, s, a, a_row, a_k, b_row, b_k, d);
    } else {
        if (p.f32) hipLaunchKernelGGL((dense_pieces_kernel<float, false>), grid, dim3(256), 0, s, a, a_row, a_k, b_row, b_k, d);
        else hipLaunchKernelGGL((dense_pieces_kernel<__bf16, false>), grid, dim3(256), 0, s, a, a_row, a_k, b_row, b_k, d);
    }
    return hipGetLastError();
}

}  // namespace alpha
