// Launchers of the dense product's tile kernel, one translation unit per storage of the operands.
#pragma once
#include "dense_gemm_kernel.hpp"

namespace alpha {

hipError_t launch_dense_tile_ss(hipStream_t s, const DenseTileArgs &a, bool big, int f32);      // both straight
hipError_t launch_dense_tile_gated(hipStream_t s, const DenseTileArgs &a, bool big, int f32);
hipError_t launch_dense_tile_st(hipStream_t s, const DenseTileArgs &a, bool big, int f32);      // B with k as its rows
hipError_t launch_dense_tile_tt(hipStream_t s, const DenseTileArgs &a, bool big, int f32);      // both with k as their rows

template <typename T, bool AT, bool BT, DenseOut OUT, int BM, int BN, int WM, int WN>
inline hipError_t launch_dense_tile(hipStream_t s, const DenseTileArgs &a)
{
    constexpr size_t lds = 4 * (BM + BN) * 64;
    const hipError_t e = ensure_dynamic_lds<dense_tile_kernel<T, AT, BT, OUT, BM, BN, WM, WN>>(lds);
    if (e != hipSuccess) return e;
    const unsigned blocks = (unsigned)a.tiles_m * (unsigned)a.tiles_n * (unsigned)a.split;
    hipLaunchKernelGGL((dense_tile_kernel<T, AT, BT, OUT, BM, BN, WM, WN>), dim3(blocks), dim3(WM * WN * 64), lds, s, a);
    return hipGetLastError();
}

// the output's kind and the tile's shape at run time
template <bool AT, bool BT, DenseOut WHOLE, DenseOut PIECES>
inline hipError_t launch_dense_tile_any(hipStream_t s, const DenseTileArgs &a, bool big, int f32)
{
    if (big) {
        if (a.split > 1) return launch_dense_tile<float, AT, BT, PIECES, 256, 256, 2, 4>(s, a);
        return f32 ? launch_dense_tile<float, AT, BT, WHOLE, 256, 256, 2, 4>(s, a) : launch_dense_tile<__bf16, AT, BT, WHOLE, 256, 256, 2, 4>(s, a);
    }
    if (a.split > 1) return launch_dense_tile<float, AT, BT, PIECES, 128, 128, 2, 2>(s, a);
    return f32 ? launch_dense_tile<float, AT, BT, WHOLE, 128, 128, 2, 2>(s, a) : launch_dense_tile<__bf16, AT, BT, WHOLE, 128, 128, 2, 2>(s, a);
}

}  // namespace alpha
