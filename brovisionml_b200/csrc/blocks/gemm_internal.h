// Between the planning of a matrix product (gemm.cu) and its kernels.
#pragma once

#include <cuda.h>

#include "blocks_internal.h"

namespace bvml {
namespace blocks {

struct TileMaps {
    CUtensorMap a[2];  // one a segment
    CUtensorMap b[2];  // one a segment, or gate and up
    CUtensorMap o[2];  // out, out2: boxes of 32 rows x 128 bytes
};

// Division of n < 2^31 by d >= 2: n / d = (n mul >> 32) >> shift with 2^shift < d <=
// 2^(shift + 1) and mul = ceil(2^(32 + shift) / d). mul d exceeds 2^(32 + shift) by
// less than d, so n times the excess stays below 2^(32 + shift): the quotient is exact.
struct Division {
    uint32_t mul, shift;
};

inline Division divide_by(uint32_t d) {
    Division v{0, 0};
    if (d < 2) return v;  // not used: see work_of
    while ((uint64_t)2 << v.shift < d) ++v.shift;
    v.mul = (uint32_t)((((uint64_t)1 << (32 + v.shift)) + d - 1) / d);
    return v;
}

// TileArgs::vec
enum : int {
    kOn16 = 1,     // few rows: every row and every vector over columns starts on 16 bytes (for
                   // the tiles always, and an output's row ends there)
    kWideSave = 2  // save's on 32
};

struct TileArgs {
    int M, N;              // output rows and columns (features when gated)
    int steps[2];          // K steps of each segment
    int tiles_m, tiles_n;
    int splits;            // shares of K, each a work item of its own
    uint32_t idesc;
    int group;                    // 2^group tile rows are walked together
    Division by_tiles, by_group;  // tiles_m * tiles_n, 2^group * tiles_n
    const float* row_scale;
    const float* col_scale[2];
    const float* bias;
    const void* residual;
    void* out;
    void* out2;
    void* save[2];
    long long ldr, ldo, ldo2, lds[2];
    int rows0, rows1;
    int out_rows;  // rows of out, and of out2 where there is one
    int out_type, act, vec;
    uint32_t wait_limit;  // attempts of a wait between the kernel's roles (gemm_wait_limit)
    float* slab;  // splits > 1: (splits, M, ldslab) fp32 partial sums
    long long ldslab;
};

// bn: the pair's columns (256, 192, 128 or 64; gated or with B transposed: 256 or 128)
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
