// Launchers of the feed-forward operators (libbvml_blocks.so), between the C
// entry points (blocks_api.cu) and the kernels.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "bvml_blocks.h"

namespace bvml {
namespace blocks {

inline size_t elem_size(int type) { return type == BVML_F32 ? 4 : type == BVML_E4M3 ? 1 : 2; }
inline size_t round256(size_t n) { return (n + 255) & ~size_t(255); }
inline bool on16(const void* p, long long ld, size_t es) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ((size_t)ld * es & 15) == 0;
}

// SMs of the current device.
cudaError_t sm_count(int* sms);

// ------------------------------------------------------------------ RMS norm
struct NormLaunch {
    const void *x, *r, *w;  // r: residual, or null
    void *y, *sum;          // sum: null without a residual
    float* scale;           // e4m3 output only
    long long ldx, ldr, ldy, lds;
    int T, K, type, wtype;
    float eps;
};
cudaError_t launch_rms_norm(const NormLaunch& L, cudaStream_t s);

struct NormBackwardLaunch {
    const void *dy, *s, *w, *ds;  // ds: null without one
    void *dx, *dw;
    float* partial;  // norm_backward_parts(T) x K
    long long lddy, lds, ldds, lddx;
    int T, K, type, wtype;
    float eps;
};
int norm_backward_parts(int T, int K);
cudaError_t launch_rms_norm_backward(const NormBackwardLaunch& L, cudaStream_t s);

// out[c] = sum over rows of part[row * cols + c], in a fixed order; out of `type`
cudaError_t launch_column_sum(const float* part, int rows, int cols, void* out, int type,
                              cudaStream_t s);

// ---------------------------------------------------------- matrix products
// D[m, n] = sum over the segments i and k < k[i] of A_i[m, k] B_i[n, k], then
// the epilogue. A_i is stored (M, k) with row stride lda, or, with a_t, (k, M);
// B_i (N, k), or (k, N) with b_t. Gated: two products with the same A over one
// segment, B_0 the gate's and B_1 the up projection's weights.
struct GemmLaunch {
    const void* a[2];
    const void* b[2];
    long long lda[2], ldb[2];
    int k[2];  // k[1] = 0: one segment (and always when gated)
    bool a_t, b_t, gated;
    int M, N;
    int in_type, out_type, act;
    const float* row_scale;     // (M) or null
    const float* col_scale[2];  // (N) each or null; [1] when gated
    const float* bias;          // (N) or null
    const void* residual;       // (M, N) of out_type or null
    void* out;                  // (M, N)
    void* save[2];              // z, or g and u; null: not kept
    long long ldr, ldo, lds[2];
    // rows >= rows1 go to out2 as row - rows1, rows in [rows0, rows1) nowhere
    // (out2 null: every row to out)
    void* out2;
    long long ldo2;
    int rows0, rows1;
};
// Scratch bytes, none for operands on 16-byte rows and enough tiles to go round.
size_t gemm_workspace_bytes(const GemmLaunch& L);
cudaError_t launch_gemm(const GemmLaunch& L, void* workspace, cudaStream_t s);
// 0, or what a bounded wait that gave up recorded; resets it (synchronous).
cudaError_t gemm_errors(int* word);
// Attempts of each wait between a kernel's roles for the launches that follow, in every
// thread; returns those before. Waits for what is in flight keep a limit of their own.
uint32_t gemm_wait_limit(uint32_t attempts);

// -------------------------------------------------- the products' derivatives
// dz = dy act'(z) (T, N) of `type` into dz (row stride lddz) unless dz is null,
// and column sums of dz before rounding into partial (act_backward_parts x N)
// unless that is null.
struct ActBackwardLaunch {
    const void *dy, *z;
    void* dz;
    float* partial;
    long long lddy, ldz, lddz;
    int T, N, type, act;
};
int act_backward_parts(int T, int N);
cudaError_t launch_act_backward(const ActBackwardLaunch& L, cudaStream_t s);
// dg = dh u act'(g), du = dh act(g)
struct GatedBackwardLaunch {
    const void *dh, *g, *u;
    void *dg, *du;
    long long lddh, ldg, ldu, ldd;
    int T, F, type, act;
};
cudaError_t launch_gated_backward(const GatedBackwardLaunch& L, cudaStream_t s);

}  // namespace blocks
}  // namespace bvml
