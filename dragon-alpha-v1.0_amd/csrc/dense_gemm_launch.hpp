// Launchers of the dense products' tile kernels, one translation unit per storage of the operands.
#pragma once
#include "dense_gemm_f32_kernel.hpp"
#include "dense_gemm_kernel.hpp"

namespace alpha {

// The tile shapes: 256 x 256 (eight wavefronts, two by four; bf16 only), 256 x 128 (four by two), 128 x 128 (bf16 four
// wavefronts, fp32 eight: 10 % faster than four, whose waits nothing fills).
// LDS, bf16: a ring of four buffers, 128, 96 and 64 KB, so two workgroups of the last share a compute unit; fp32: two buffers of
// three planes, 144 and 96 KB.
enum DenseTile { DENSE_TILE_256, DENSE_TILE_256_128, DENSE_TILE_128, DENSE_TILES };
constexpr int DENSE_TILE_M[DENSE_TILES] = {256, 256, 128}, DENSE_TILE_N[DENSE_TILES] = {256, 128, 128};

hipError_t launch_dense_tile_ss(hipStream_t s, const DenseTileArgs &a, DenseTile tile, int f32);      // both straight
hipError_t launch_dense_tile_gated(hipStream_t s, const DenseTileArgs &a, DenseTile tile, int f32);
hipError_t launch_dense_tile_st(hipStream_t s, const DenseTileArgs &a, DenseTile tile, int f32);      // B with k as its rows
hipError_t launch_dense_tile_tt(hipStream_t s, const DenseTileArgs &a, DenseTile tile, int f32);      // both with k as their rows

template <auto KERNEL>
inline hipError_t launch_dense_tile(hipStream_t s, const DenseTileArgs &a, int threads, size_t lds)
{
    const hipError_t e = ensure_dynamic_lds<KERNEL>(lds);
    if (e != hipSuccess) return e;
    const unsigned blocks = (unsigned)a.whole + ((unsigned)a.tiles_m * (unsigned)a.tiles_n - (unsigned)a.whole) * (unsigned)a.split;
    hipLaunchKernelGGL(KERNEL, dim3(blocks), dim3(threads), lds, s, a);
    return hipGetLastError();
}

// the operands' type and the tile's shape at run time
template <bool AT, bool BT, bool GATED>
inline hipError_t launch_dense_tile_any(hipStream_t s, const DenseTileArgs &a, DenseTile tile, int f32)
{
    if (f32) {
        if (tile == DENSE_TILE_256_128) return launch_dense_tile<dense_tile_f32_kernel<AT, BT, GATED, 256, 128, 4, 2>>(s, a, 512, 2 * 3 * (256 + 128) * 64);
        return launch_dense_tile<dense_tile_f32_kernel<AT, BT, GATED, 128, 128, 4, 2>>(s, a, 512, 2 * 3 * (128 + 128) * 64);
    }
    switch (tile) {
    case DENSE_TILE_256: return launch_dense_tile<dense_tile_kernel<AT, BT, GATED, 256, 256, 2, 4, 4>>(s, a, 512, 4 * (256 + 256) * 64);
    case DENSE_TILE_256_128: return launch_dense_tile<dense_tile_kernel<AT, BT, GATED, 256, 128, 4, 2, 4>>(s, a, 512, 4 * (256 + 128) * 64);
    default: return launch_dense_tile<dense_tile_kernel<AT, BT, GATED, 128, 128, 2, 2, 4>>(s, a, 256, 4 * (128 + 128) * 64);
    }
}

}  // namespace alpha
