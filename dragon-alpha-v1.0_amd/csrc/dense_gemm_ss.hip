// The tile kernel for both operands with k along their rows (forward).
#include "dense_gemm_launch.hpp"

namespace alpha {

hipError_t launch_dense_tile_ss(hipStream_t s, const DenseTileArgs &a, DenseTile tile, int f32)
{
    return launch_dense_tile_any<false, false, false>(s, a, tile, f32);
}

}  // namespace alpha
