// Forward products on 16-bit operands (gemm_tile.cuh).
#include "gemm_tile.cuh"

namespace bvml {
namespace blocks {

cudaError_t launch_tile_nt(int bn, bool gated, const TileMaps& m, const TileArgs& a, int pairs,
                           cudaStream_t s) {
    if (gated) {
        if (bn == 256) return launch_tile<256, false, false, false, true>(m, a, pairs, s);
        return launch_tile<128, false, false, false, true>(m, a, pairs, s);
    }
    if (bn == 256) return launch_tile<256, false, false, false, false>(m, a, pairs, s);
    if (bn == 192) return launch_tile<192, false, false, false, false>(m, a, pairs, s);
    if (bn == 128) return launch_tile<128, false, false, false, false>(m, a, pairs, s);
    return launch_tile<64, false, false, false, false>(m, a, pairs, s);
}

BVML_TILE_ERROR_READER(tile_nt_error)

}  // namespace blocks
}  // namespace bvml
