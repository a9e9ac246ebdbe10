// Launchers of the dense product's tile kernel, one translation unit per storage of the operands.
#pragma once
#include "dense_gemm_kernel.hpp"

namespace alpha {

// The tile shapes: 256 x 256 (eight wavefronts, two by four), 256 x 128 (four by two), 128 x 128 (four wavefronts), each a
// ring of four buffers: 128, 96 and 64 KB of LDS, so two workgroups of the last share a compute unit.
enum DenseTile { DENSE_TILE_256, DENSE_TILE_256_128, DENSE_TILE_128, DENSE_TILES };
constexpr int DENSE_TILE_M[DENSE_TILES] = {256, 256, 128}, DENSE_TILE_N[DENSE_TILES] = {256, 128, 128};

hipError_t launch_dense_tile_ss(hipStream_t s, const DenseTileArgs &a, DenseTile tile, int f32);      // both straight
hipError_t launch_dense_tile_gated(hipStream_t s, const DenseTileArgs &a, DenseTile tile, int f32);
hipError_t launch_dense_tile_st(hipStream_t s, const DenseTileArgs &a, DenseTile tile, int f32);      // B with k as its rows
hipError_t launch_dense_tile_tt(hipStream_t s, const DenseTileArgs &a, DenseTile tile, int f32);      // both with k as their rows

template <typename T, bool AT, bool BT, bool GATED, int BM, int BN, int WM, int WN>
inline hipError_t launch_dense_tile(hipStream_t s, const DenseTileArgs &a)
{
    constexpr int stages = 4;
    constexpr size_t lds = stages * (BM + BN) * 64;
    constexpr auto kernel = dense_tile_kernel<T, AT, BT, GATED, BM, BN, WM, WN, stages>;
    const hipError_t e = ensure_dynamic_lds<kernel>(lds);
    if (e != hipSuccess) return e;
    const unsigned blocks = (unsigned)a.whole + ((unsigned)a.tiles_m * (unsigned)a.tiles_n - (unsigned)a.whole) * (unsigned)a.split;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(WM * WN * 64), lds, s, a);
    return hipGetLastError();
}

// the output's type and the tile's shape at run time
template <bool AT, bool BT, bool GATED>
inline hipError_t launch_dense_tile_any(hipStream_t s, const DenseTileArgs &a, DenseTile tile, int f32)
{
    switch (tile) {
    case DENSE_TILE_256: return f32 ? launch_dense_tile<float, AT, BT, GATED, 256, 256, 2, 4>(s, a) : launch_dense_tile<__bf16, AT, BT, GATED, 256, 256, 2, 4>(s, a);
    case DENSE_TILE_256_128: return f32 ? launch_dense_tile<float, AT, BT, GATED, 256, 128, 4, 2>(s, a) : launch_dense_tile<__bf16, AT, BT, GATED, 256, 128, 4, 2>(s, a);
    default: return f32 ? launch_dense_tile<float, AT, BT, GATED, 128, 128, 2, 2>(s, a) : launch_dense_tile<__bf16, AT, BT, GATED, 128, 128, 2, 2>(s, a);
    }
}

}  // namespace alpha
