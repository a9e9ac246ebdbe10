// The tile kernel for both operands with k as their rows (deltaW).
#include "dense_gemm_launch.hpp"

namespace alpha {

hipError_t launch_dense_tile_tt(hipStream_t s, const DenseTileArgs &a, DenseTile tile, int f32)
{
    return launch_dense_tile_any<true, true, false>(s, a, tile, f32);
}

}  // namespace alpha
