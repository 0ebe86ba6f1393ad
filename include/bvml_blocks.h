/*
 * bvml_blocks.h -- C ABI of the feed-forward operators (libbvml_blocks.so,
 * built from brovisionml_b200/csrc/blocks/): RMS norm, linear and gated linear
 * over rows of features, with their backward passes. A library of its own
 * beside libbvml_dsine.so, whose ABI stays as it is; no counterpart in the
 * reference, which has no training and no such layer.
 *
 * Conventions (as in bvml_dsine.h, whose status codes are used)
 *  - All pointers are DEVICE pointers of the current CUDA device. A matrix is
 *    a pointer and a row stride `ld` in elements (>= the columns); its last
 *    axis is contiguous. Pointers are aligned to their element. Rows that
 *    start on 16 bytes (pointer and stride) are read in place; others are
 *    accepted and laid out anew in the workspace first, as are vectors over
 *    output features (bias, scales) that do not. Outputs of the
 *    products whose rows do not start and end on 16 bytes likewise go through
 *    the workspace. The *_workspace_bytes calls look at the pointers'
 *    alignment, so they take the arguments of the call itself.
 *  - A dimension is at most 2^30 - 64.
 *  - Types: BVML_F32, BVML_F16 (bvml_dsine.h), BVML_BF16, BVML_E4M3. Sums and
 *    statistics are 32-bit; results are rounded once, to nearest.
 *  - `stream` is a cudaStream_t (NULL = the legacy default stream). Calls are
 *    asynchronous, allocate nothing and can be captured into a CUDA graph.
 *  - An output may not overlap an input or another output (checked).
 *  - T = 0 rows are fine: the products' weight gradients are then zeros.
 *  - Workspaces are scratch: 256-byte aligned, their content before a call
 *    does not matter and after it is unspecified; two calls (or captured
 *    graphs) that may overlap on the GPU need one each.
 *  - Every call returns BVML_OK or a BVML_E* code and never throws; the text
 *    of the calling thread's last failure here is bvml_blocks_last_error(),
 *    "dsine ops: ..." for arguments, "dsine cuda: ..." for CUDA failures.
 */
#ifndef BVML_BLOCKS_H
#define BVML_BLOCKS_H

#include "bvml_dsine.h"

#ifdef __cplusplus
extern "C" {
#endif

#define BVML_BLOCKS_VERSION 1

/* element types beside bvml_dtype's */
#define BVML_BF16 2
#define BVML_E4M3 3 /* 8-bit floats, four exponent and three fraction bits, largest value 448 */

/* bad workspace: none or too small a one was given, or not 256-byte aligned */
#define BVML_EWORKSPACE 4

/* activations: 0 to 3 as in bvml_conv2d_nhwc_f16 */
#define BVML_ACT_NONE 0
#define BVML_ACT_RELU 1
#define BVML_ACT_SIGMOID 2
#define BVML_ACT_TANH 3
#define BVML_ACT_SILU 4 /* z sigmoid(z) */
#define BVML_ACT_GELU 5 /* z Phi(z), Phi the normal distribution function (erf form) */
/* sigmoid, Phi and their derivatives are zero where they are below 2^-126 */

const char* bvml_blocks_last_error(void);
int bvml_blocks_version(void);

/*
 * Waits inside the matrix-product kernels are bounded; one that gives up (the
 * GPU stopped making progress) is recorded per device instead of hanging, and
 * the results of that call are unspecified. Synchronises `stream`, returns
 * BVML_OK, or BVML_ECUDA once for what was recorded since the last call. Not for a
 * stream that is being captured.
 */
int bvml_blocks_status(void* stream);
/*
 * Attempts of each wait between a matrix product's copies, MMAs and epilogue, for the
 * launches of the process that follow; returns the value before (4194304 at first). For tests of that
 * path: with 1 (or 0) a wait gives up where what it waits for is not there yet. What is in
 * flight then is waited for all the same before the kernel leaves.
 */
unsigned bvml_blocks_wait_limit(unsigned attempts);

/*
 * s = x + residual (residual may be NULL: s = x), y = s / sqrt(mean(s^2) + eps) * weight,
 * row by row over K features. The norm is taken of the sum before it is
 * rounded; `sum` (may be NULL without a residual) gets s rounded to `dtype`.
 *   x, residual, y, sum (T, K) of `dtype` (F32, F16 or BF16); weight (K) of weight_dtype:
 *   F32, or `dtype`. A row with NaN gives NaN; eps >= 0.
 */
int bvml_rms_norm(const void* x, long long ldx, const void* residual, long long ldr,
                  const void* weight, int T, int K, int dtype, int weight_dtype, float eps,
                  void* y, long long ldy, void* sum, long long lds, void* stream);

/*
 * bvml_rms_norm with y in 8 bits: scale[t] = max_k |y[t, k]| / 448 (fp32),
 * q[t, k] = y[t, k] / scale[t] rounded to nearest e4m3, so y ~ q * scale. A row whose
 * largest |y| is below 2^-110 counts as zeros: q = 0, scale = 1. A row with NaN or
 * infinities in s or y (zeros with eps = 0 are 0 / 0) has a NaN scale. `q` (T, K) e4m3.
 */
int bvml_rms_norm_e4m3(const void* x, long long ldx, const void* residual, long long ldr,
                       const void* weight, int T, int K, int dtype, int weight_dtype, float eps,
                       void* q, long long ldq, float* scale, void* sum, long long lds,
                       void* stream);

/*
 * Backward of bvml_rms_norm for dy and, when the sum went on as the residual
 * stream, its gradient dsum (NULL: none): with r = 1 / sqrt(mean(s^2) + eps), n = s r,
 *   dx = r (dy w - n mean(dy w n)) + dsum    (the gradient of x and of the residual)
 *   dweight = sum_t dy n                      (weight_dtype; sums in 32 bits, in a
 *                                              fixed order: runs agree bit for bit)
 * s (T, K): the sum that the forward pass gave, or x without a residual.
 */
size_t bvml_rms_norm_backward_workspace_bytes(int T, int K);
int bvml_rms_norm_backward(const void* dy, long long lddy, const void* s, long long lds,
                           const void* weight, const void* dsum, long long ldds, int T, int K,
                           int dtype, int weight_dtype, float eps, void* dx, long long lddx,
                           void* dweight, void* workspace, size_t workspace_bytes, void* stream);

/*
 * y = act(z) + residual with z = x w^T + bias: x (T, K), w (N, K), y and
 * residual (T, N); fp32 accumulation on the tensor cores.
 *   in_type F16 or BF16 (x and w alike), out_type the same or F32; or in_type
 *   E4M3 with x_scale (T) and w_scale (N) fp32, the value of x[t, k] being
 *   x[t, k] x_scale[t], and out_type F16, BF16 or F32. The sum is multiplied by
 *   x_scale[t] w_scale[n], one fp32 number: it has to be within fp32's normal range.
 *   bias (N) fp32 or NULL; residual of out_type or NULL; z, when not NULL,
 *   gets the pre-activation in out_type (the backward pass takes it).
 */
typedef struct {
    const void* x;
    const void* w;
    const float* x_scale; /* E4M3 inputs only */
    const float* w_scale;
    const float* bias;
    const void* residual;
    void* y;
    void* z;
    long long ldx, ldw, ldr, ldy, ldz;
    int T, K, N;
    int in_type, out_type, act;
} bvml_linear_args;
size_t bvml_linear_workspace_bytes(const bvml_linear_args* a);
int bvml_linear(const bvml_linear_args* a, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Backward of bvml_linear: dz = dy act'(z),
 *   dx = dz w (T, K), dw = dz^T x (N, K), dbias = sum_t dz (N, fp32; NULL: not wanted).
 * The residual's gradient is dy itself. `type` F16 or BF16 for every matrix;
 * z (T, N) may be NULL when act is BVML_ACT_NONE. dz is rounded to `type` for
 * the two products, dbias sums it before. dx or dw may be NULL (not wanted).
 */
typedef struct {
    const void* dy;
    const void* z;
    const void* x;
    const void* w;
    void* dx;
    void* dw;
    float* dbias;
    long long lddy, ldz, ldx, ldw, lddx, lddw;
    int T, K, N;
    int type, act;
} bvml_linear_backward_args;
size_t bvml_linear_backward_workspace_bytes(const bvml_linear_backward_args* a);
int bvml_linear_backward(const bvml_linear_backward_args* a, void* workspace,
                         size_t workspace_bytes, void* stream);

/*
 * h = act(g) u with g = x w_gate^T and u = x w_up^T: x (T, K), w_gate and w_up
 * (F, K), h (T, F). Types as bvml_linear (gate_scale, up_scale (F) with E4M3).
 * act: not BVML_ACT_NONE. g and u, when not NULL, get the two projections in
 * out_type (both or neither; the backward pass takes them).
 */
typedef struct {
    const void* x;
    const void* w_gate;
    const void* w_up;
    const float* x_scale;
    const float* gate_scale;
    const float* up_scale;
    void* h;
    void* g;
    void* u;
    long long ldx, ldw_gate, ldw_up, ldh, ldg, ldu;
    int T, K, F;
    int in_type, out_type, act;
} bvml_gated_args;
size_t bvml_gated_linear_workspace_bytes(const bvml_gated_args* a);
int bvml_gated_linear(const bvml_gated_args* a, void* workspace, size_t workspace_bytes,
                      void* stream);

/*
 * Backward of bvml_gated_linear: dg = dh u act'(g), du = dh act(g) (rounded to
 * `type` for the products),
 *   dx = dg w_gate + du w_up (T, K), dw_gate = dg^T x, dw_up = du^T x (F, K).
 * dx, or both of dw_gate and dw_up, may be NULL (not wanted).
 */
typedef struct {
    const void* dh;
    const void* g;
    const void* u;
    const void* x;
    const void* w_gate;
    const void* w_up;
    void* dx;
    void* dw_gate;
    void* dw_up;
    long long lddh, ldg, ldu, ldx, ldw_gate, ldw_up, lddx, lddw_gate, lddw_up;
    int T, K, F;
    int type, act;
} bvml_gated_backward_args;
size_t bvml_gated_linear_backward_workspace_bytes(const bvml_gated_backward_args* a);
int bvml_gated_linear_backward(const bvml_gated_backward_args* a, void* workspace,
                               size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* BVML_BLOCKS_H */
