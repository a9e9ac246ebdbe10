// The tile kernel for B with k as its rows (deltaX).
#include "dense_gemm_launch.hpp"

namespace alpha {

hipError_t launch_dense_tile_st(hipStream_t s, const DenseTileArgs &a, DenseTile tile, int f32)
{
    return launch_dense_tile_any<false, true, false>(s, a, tile, f32);
}

}  // namespace alpha
