// Forward products on e4m3 operands (gemm_tile.cuh).
#include "gemm_tile.cuh"

namespace bvml {
namespace blocks {

cudaError_t launch_tile_nt_f8(int bn, bool gated, const TileMaps& m, const TileArgs& a, int pairs,
                           cudaStream_t s) {
    if (gated) {
        if (bn == 256) return launch_tile<256, false, false, true, true>(m, a, pairs, s);
        return launch_tile<128, false, false, true, true>(m, a, pairs, s);
    }
    if (bn == 256) return launch_tile<256, false, false, true, false>(m, a, pairs, s);
    if (bn == 192) return launch_tile<192, false, false, true, false>(m, a, pairs, s);
    if (bn == 128) return launch_tile<128, false, false, true, false>(m, a, pairs, s);
    return launch_tile<64, false, false, true, false>(m, a, pairs, s);
}

BVML_TILE_ERROR_READER(tile_nt_f8_error)

}  // namespace blocks
}  // namespace bvml
