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
#pragma unroll 4
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
    DenseTile tile;
    int split, per, tiles_m, tiles_n, steps;
    double us;
};

// Tile shape and cut of the reduction: the least of an estimate of the device's time, its constants measured on NT products
// of 256 x 256 x 256 to 8192 x 4096 x 4096 (a workgroup's step with the device nearly empty and full, 256 / 256 x 128 / 128:
// 0.57 / 0.34 / 0.36 and 0.72 / 0.48 / 0.59 us, the last with two workgroups on a compute unit). `room`: bytes for the pieces.
Plan make_plan(int M, int N, int K, int parts, int sources, int gated, size_t room)
{
    static constexpr double empty[DENSE_TILES] = {0.57, 0.34, 0.36}, full[DENSE_TILES] = {0.72, 0.48, 0.59}, fixed[DENSE_TILES] = {6.5, 5.0, 3.0};
    const int cus = std::max(1, device_cu_count());
    const int nk = std::max(1, (K + 31) / 32), combos = (parts == 3 ? 6 : 1) * sources, steps = nk * combos;
    const double outputs = (double)M * N * (gated ? 2 : 1), bytes_per_us = 4.2e6;
    Plan best{};
    best.us = 1e30;
    for (int tile = 0; tile < DENSE_TILES; tile++) {
        const int bm = DENSE_TILE_M[tile], bn = DENSE_TILE_N[tile] / (gated ? 2 : 1);
        const int tm = (int)(((long)M + bm - 1) / bm), tn = (N + bn - 1) / bn;
        const long tiles = (long)tm * tn;
        for (int split = 1; split <= 64; split++) {
            // whole k steps: a piece holds all parts of its products, so none leaves fp32's range that the sum would not
            // (and an even number of steps: the kernel's loop does two at a time)
            const int per = (nk + 2 * split - 1) / (2 * split) * 2 * combos;
            if (split > 1 && (per < 8 || split * outputs * 4 > (double)room)) break;
            if ((steps + per - 1) / per != split) continue;   // every piece has a step
            const long groups = tiles * split;
            const bool pairs = tile == DENSE_TILE_128 && groups > cus;
            const long slots = pairs ? 2l * cus : cus, rounds = (groups + slots - 1) / slots;
            const double fill = std::min(1.0, (double)groups / slots);
            double us = 3.5 + rounds * (per * (tile == DENSE_TILE_128 ? (pairs ? full[tile] : empty[tile]) : empty[tile] + (full[tile] - empty[tile]) * fill) + fixed[tile]);
            us += split > 1 ? 5.0 + outputs * (8.0 * split + 2) / bytes_per_us : outputs * (parts == 3 ? 4 : 2) / bytes_per_us;
            if (us < best.us) best = Plan{(DenseTile)tile, split, per, tm, tn, steps, us};
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

double dense_product_us(int M, int N, int K, int parts, int sources, int gated) { return make_plan(M, N, K, parts, sources, gated, (size_t)1 << 60).us; }

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
    if (p.a_t) e = launch_dense_tile_tt(s, a, plan.tile, p.f32);
    else if (p.b_t) e = launch_dense_tile_st(s, a, plan.tile, p.f32);
    else if (p.gated) e = launch_dense_tile_gated(s, a, plan.tile, p.f32);
    else e = launch_dense_tile_ss(s, a, plan.tile, p.f32);
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
