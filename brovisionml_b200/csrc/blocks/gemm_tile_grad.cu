// The backward passes' products (gemm_tile.cuh): dx = dz w reads w with the
// contracted axis outermost, dw = dz^T x both operands.
#include "gemm_tile.cuh"

namespace bvml {
namespace blocks {

cudaError_t launch_tile_grad(int bn, bool a_t, const TileMaps& m, const TileArgs& a, int pairs,
                             cudaStream_t s) {
    if (a_t) {
        if (bn == 256) return launch_tile<256, true, true, false, false>(m, a, pairs, s);
        return launch_tile<128, true, true, false, false>(m, a, pairs, s);
    }
    if (bn == 256) return launch_tile<256, false, true, false, false>(m, a, pairs, s);
    return launch_tile<128, false, true, false, false>(m, a, pairs, s);
}

BVML_TILE_ERROR_READER(tile_grad_error)

}  // namespace blocks
}  // namespace bvml
