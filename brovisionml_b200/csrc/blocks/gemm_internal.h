// Between the planning of a matrix product (gemm.cu) and its kernels.
#pragma once

#include <cuda.h>

#include "blocks_internal.h"

namespace bvml {
namespace blocks {

struct TileMaps {
    CUtensorMap a[2];  // one a segment
    CUtensorMap b[2];  // one a segment, or gate and up
};

// groups of eight columns start on 16 bytes in ...
enum : int { kVecOut = 1, kVecOut2 = 2, kVecRes = 4, kVecSave = 8 };

struct TileArgs {
    int M, N;              // output rows and columns (features when gated)
    int steps[2];          // K steps of each segment
    int tiles_m, tiles_n;
    int splits;            // shares of K, each a work item of its own
    uint32_t idesc;
    const float* row_scale;
    const float* col_scale[2];
    const float* bias;
    const void* residual;
    void* out;
    void* out2;
    void* save[2];
    long long ldr, ldo, ldo2, lds[2];
    int rows0, rows1;
    int out_type, act, vec;
    float* slab;  // splits > 1: (splits, M, ldslab) fp32 partial sums
    long long ldslab;
};

// bn: the pair's columns (256, 128 or 64; transposed B: at least 128)
cudaError_t launch_tile_nt(int bn, bool gated, const TileMaps& m, const TileArgs& a, int pairs,
                           cudaStream_t s);
cudaError_t launch_tile_nt_f8(int bn, bool gated, const TileMaps& m, const TileArgs& a, int pairs,
                              cudaStream_t s);
cudaError_t launch_tile_grad(int bn, bool a_t, const TileMaps& m, const TileArgs& a, int pairs,
                             cudaStream_t s);

// Few rows: weights as the MMA's rows, tokens as its columns, K shared out over
// a cluster of `split` CTAs. tok: columns a CTA takes (16, 32, 64 or 128).
// maps: a[0] the tokens', b[0] and b[1] the weights'.
struct SkinnyArgs {
    TileArgs t;     // steps[0], the epilogue
    int split;      // 1, 2, 4 or 8, at most steps[0]
};
cudaError_t launch_skinny(int tok, bool f8, bool gated, const TileMaps& m, const SkinnyArgs& a,
                          cudaStream_t s);
cudaError_t skinny_error(int* word);

cudaError_t tile_nt_error(int* word);
cudaError_t tile_nt_f8_error(int* word);
cudaError_t tile_grad_error(int* word);

}  // namespace blocks
}  // namespace bvml
