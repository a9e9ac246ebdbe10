// The tile kernel for the gated pair of products (forward).
#include "dense_gemm_launch.hpp"

namespace alpha {

hipError_t launch_dense_tile_gated(hipStream_t s, const DenseTileArgs &a, DenseTile tile, int f32)
{
    return launch_dense_tile_any<false, false, true>(s, a, tile, f32);
}

}  // namespace alpha
