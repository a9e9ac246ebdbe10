// Launch of the dense product: tile shape and cut of the reduction by size, the second kernel that adds the pieces.
#include "dense_gemm_launch.hpp"

#include <algorithm>

namespace alpha {

// Adds the pieces of the cut tiles in their order and applies the epilogue: eight columns a thread, a workgroup 256 / (BN / 8)
// rows of a tile (gated: BN / 16 threads a row, eight columns of each filter).
template <typename T, bool GATED, bool FULL>
__global__ __launch_bounds__(256) void dense_pieces_kernel(const DenseTileArgs a, int bm, int bn)
{
    const int lanes = bn / (GATED ? 16 : 8), rows = 256 / lanes, per_tile = bm / rows;
    const int cut = (int)blockIdx.x / per_tile, row = (int)blockIdx.x % per_tile * rows + (int)threadIdx.x / lanes, lane = (int)threadIdx.x % lanes;
    int tm, tn;
    tile_at(a.whole + cut, a.tiles_m, a.tiles_n, tm, tn);
    const long m = (long)tm * bm + row;
    const int n = tn * (GATED ? bn / 2 : bn) + lane * 8;
    if (m >= a.M || n >= a.N) return;
    float v[8], u[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = u[e] = 0.f;
    // gated: of every 64 columns of a tile 32 are the gate's, the other 32 the other filter's
    const float *src = a.pieces + ((long)cut * bm + row) * bn + (GATED ? lane / 4 * 64 + lane % 4 * 8 : lane * 8);
    const long step = ((long)a.tiles_m * a.tiles_n - a.whole) * bm * bn;
#pragma unroll 4
    for (int p = 0; p < a.split; p++, src += step) {
        float t[8];
        run_load(src, t);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] += t[e];
        if constexpr (GATED) {
            run_load(src + 32, t);
#pragma unroll
            for (int e = 0; e < 8; e++) u[e] += t[e];
        }
    }
    if (a.ep.vec && n + 8 <= a.N) {
        if constexpr (GATED) dense_finish_gated<T, 8, true>(a.ep, v, u, m, n);
        else dense_finish<T, 8, FULL, true>(a.ep, v, m, n);
    } else {
        const int left = a.N - n < 8 ? a.N - n : 8;
        if constexpr (GATED) dense_finish_gated<T, 8, false>(a.ep, v, u, m, n, left);
        else dense_finish<T, 8, FULL, false>(a.ep, v, m, n, left);
    }
}

namespace {

struct Plan {
    DenseTile tile;
    int tiles_m, tiles_n, whole, split, per, steps;
    double us;
};

size_t piece_bytes(const Plan &p) { return ((size_t)p.tiles_m * p.tiles_n - p.whole) * p.split * DENSE_TILE_M[p.tile] * DENSE_TILE_N[p.tile] * 4; }

// Tile shape and cut: whole tiles for as many rounds as the device's workgroup slots go into, and the tiles that are left (or
// all, where there are few) with their reduction cut so that they fill the device once more. The choice is the least of an
// estimate of the device's time; its constants were measured on products of 256 x 256 x 256 to 8192 x 4096 x 4096: a
// workgroup's step with the device nearly empty and full, bf16 (256 / 256 x 128 / 128) 0.57 / 0.34 / 0.30 and 0.70 / 0.48 /
// 0.54 us, the last with two workgroups on a compute unit; fp32 (256 x 128 / 128) 2.05 / 1.3 and 2.55 / 1.5.
Plan make_plan(int M, int N, int K, int f32, int sources, int gated, size_t room)
{
    static constexpr double empty[2][DENSE_TILES] = {{0.57, 0.34, 0.30}, {0, 2.05, 1.3}}, full[2][DENSE_TILES] = {{0.70, 0.48, 0.54}, {0, 2.55, 1.5}};
    static constexpr double fixed[DENSE_TILES] = {6.5, 5.0, 3.0};
    const int cus = std::max(1, device_cu_count());
    const int nk = std::max(1, (K + 31) / 32), steps = nk * sources;
    const double bytes_per_us = 4.2e6, outputs = (double)M * N * (gated ? 2 : 1);
    Plan best{};
    best.us = 1e30;
    for (int t = f32 ? DENSE_TILE_256_128 : DENSE_TILE_256; t < DENSE_TILES; t++) {
        const int bm = DENSE_TILE_M[t], bn = DENSE_TILE_N[t];
        Plan p{};
        p.tile = (DenseTile)t;
        p.tiles_m = (int)(((long)M + bm - 1) / bm);
        p.tiles_n = (N * (gated ? 2 : 1) + bn - 1) / bn;
        p.steps = steps;
        const long tiles = (long)p.tiles_m * p.tiles_n;
        const double e = empty[f32 ? 1 : 0][t], f = full[f32 ? 1 : 0][t];
        const bool shared = t == DENSE_TILE_128 && !f32;     // two workgroups on a compute unit
        // time of `groups` workgroups of `per` steps each
        auto rounds_us = [&](long groups, int per) {
            const bool pairs = shared && groups > cus;
            const long slots = pairs ? 2l * cus : cus, rounds = (groups + slots - 1) / slots;
            const double filled = std::min(1.0, (double)groups / slots);
            return rounds * (per * (shared ? (pairs ? f : e) : e + (f - e) * filled) + fixed[t]);
        };
        auto consider = [&](long whole, int split) {
            // (an even number of steps: the kernels' loops do two at a time)
            p.whole = (int)whole;
            p.split = split;
            p.per = (nk + 2 * split - 1) / (2 * split) * 2 * sources;
            const long left = tiles - whole;
            p.us = 3.5 + outputs * (f32 ? 4 : 2) / bytes_per_us + (whole > 0 ? rounds_us(whole, steps) : 0.0);
            if (left > 0) {
                if (split < 2 || p.per < (f32 ? 2 : 8) || (steps + p.per - 1) / p.per != split || piece_bytes(p) > room) return;   // (every piece has a step)
                p.us += rounds_us(left * split, p.per) + 2.0 + piece_bytes(p) * 2.0 / bytes_per_us;
            }
            if (p.us < best.us) best = p;
        };
        consider(tiles, 1);
        const long slots = shared ? 2l * cus : cus, starts[2] = {0, tiles / slots * slots};
        for (int i = 0; i < 2; i++) {
            if ((i == 1 && starts[1] == 0) || starts[i] == tiles || tiles - starts[i] > slots) continue;
            for (int split = 2; split <= 64; split += split < 8 ? 1 : split < 16 ? 2 : 8) consider(starts[i], split);
        }
    }
    return best;
}

}  // namespace

size_t dense_product_piece_bytes(int M, int N, int K, int f32, int sources, int gated)
{
    // as many pieces as the plan without a limit takes
    return piece_bytes(make_plan(M, N, K, f32, sources, gated, (size_t)1 << 60));
}

double dense_product_us(int M, int N, int K, int f32, int sources, int gated) { return make_plan(M, N, K, f32, sources, gated, (size_t)1 << 60).us; }

hipError_t launch_dense_product(hipStream_t s, const DenseProduct &p)
{
    if (p.M <= 0 || p.N <= 0) return hipSuccess;
    const Plan plan = make_plan(p.M, p.N, p.K, p.f32, p.sources, p.gated, p.pieces ? p.piece_bytes : 0);
    DenseTileArgs a{};
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
    a.steps = plan.steps;
    a.whole = plan.whole;
    a.split = plan.split;
    a.per = plan.per;
    a.tiles_m = plan.tiles_m;
    a.tiles_n = plan.tiles_n;
    a.ep = p.ep;
    a.pieces = p.pieces;
    hipError_t e;
    if (p.a_t) e = launch_dense_tile_tt(s, a, plan.tile, p.f32);
    else if (p.b_t) e = launch_dense_tile_st(s, a, plan.tile, p.f32);
    else if (p.gated) e = launch_dense_tile_gated(s, a, plan.tile, p.f32);
    else e = launch_dense_tile_ss(s, a, plan.tile, p.f32);
    const int bm = DENSE_TILE_M[plan.tile], bn = DENSE_TILE_N[plan.tile], cut = plan.tiles_m * plan.tiles_n - plan.whole;
    if (e != hipSuccess || cut == 0) return e;
    const dim3 grid((unsigned)cut * (unsigned)(bm * bn / (p.gated ? 16 : 8) / 256));
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, bm, bn); };
    if (p.gated) p.f32 ? launch(dense_pieces_kernel<float, true, true>) : launch(dense_pieces_kernel<__bf16, true, true>);
    else if (p.b_t) p.f32 ? launch(dense_pieces_kernel<float, false, false>) : launch(dense_pieces_kernel<__bf16, false, false>);
    else p.f32 ? launch(dense_pieces_kernel<float, false, true>) : launch(dense_pieces_kernel<__bf16, false, true>);
    return hipGetLastError();
}

}  // namespace alpha
