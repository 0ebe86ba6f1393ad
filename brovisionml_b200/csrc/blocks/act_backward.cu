// The elementwise half of the products' backward passes:
//   linear  dz = dy act'(z), and the bias gradient's sums over rows of dz
//   gated   dg = dh u act'(g), du = dh act(g)
//
// Bound by HBM: each input is read once, 16 bytes a thread and access; a block
// covers 256 columns and walks rows, a thread keeps eight columns' sums in
// registers. The sums over a block's warps and over blocks run in a fixed
// order. What the matrix products read back (dz, dg, du) is rounded to 16 bits,
// the type the tensor cores take; the bias gradient sums the 32-bit values.
#include "blocks_common.cuh"
#include "blocks_internal.h"

namespace bvml {
namespace blocks {
namespace {

constexpr int kCols = 256;  // columns of a block: 32 lanes of eight
constexpr int kRowThreads = 8;

// Up to eight columns c .. of row pointer p as floats, zeros past n.
template <typename T>
__device__ __forceinline__ void load_cols(const T* p, int c, int n, bool vec, float (&v)[8]) {
    if (vec && c + 8 <= n) {
        load8(p + c, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < n ? to_f(p[c + e]) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store_cols(T* p, int c, int n, bool vec, const float (&v)[8]) {
    if (vec && c + 8 <= n) {
        store8(p + c, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < n) p[c + e] = from_f<T>(v[e]);
    }
}

template <typename T>
__global__ void __launch_bounds__(kCols)
act_backward_kernel(const ActBackwardLaunch L, bool vec_dy, bool vec_z, bool vec_dz) {
    __shared__ float sh[kRowThreads][kCols];
    const int lane = threadIdx.x % 32, ry = threadIdx.x / 32;
    const int c = blockIdx.x * kCols + lane * 8;
    float sum[8] = {};
    for (long long t = (long long)blockIdx.y * kRowThreads + ry; t < L.T;
         t += (long long)gridDim.y * kRowThreads) {
        if (c >= L.N) break;
        float d[8];
        load_cols(static_cast<const T*>(L.dy) + t * L.lddy, c, L.N, vec_dy, d);
        if (L.z) {
            float z[8];
            load_cols(static_cast<const T*>(L.z) + t * L.ldz, c, L.N, vec_z, z);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float f, g;
                act_grad_f(z[e], L.act, f, g);
                d[e] *= g;
            }
        }
        if (L.dz) store_cols(static_cast<T*>(L.dz) + t * L.lddz, c, L.N, vec_dz, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += c + e < L.N ? d[e] : 0.0f;
    }
    if (!L.partial) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) sh[ry][lane * 8 + e] = sum[e];
    __syncthreads();
    const int n = blockIdx.x * kCols + threadIdx.x;
    if (n < L.N) {
        float v = sh[0][threadIdx.x];
#pragma unroll
        for (int i = 1; i < kRowThreads; ++i) v += sh[i][threadIdx.x];
        L.partial[(long long)blockIdx.y * L.N + n] = v;
    }
}

// g, u <- dh u act'(g), dh act(g); the activation is chosen outside the loops
__device__ __forceinline__ void grad_rows(int act, const float (&dh)[2][8], float (&g)[2][8],
                                          float (&u)[2][8]) {
    switch (act) {
#define BVML_GRAD_ROWS(code)                                  \
    case code:                                                \
        _Pragma("unroll") for (int i = 0; i < 2; ++i)         \
            _Pragma("unroll") for (int e = 0; e < 8; ++e) {   \
                float f, d;                                   \
                act_grad_f(g[i][e], code, f, d);              \
                g[i][e] = dh[i][e] * u[i][e] * d;             \
                u[i][e] = dh[i][e] * f;                       \
            }                                                 \
        break;
        BVML_GRAD_ROWS(BVML_ACT_RELU)
        BVML_GRAD_ROWS(BVML_ACT_SIGMOID)
        BVML_GRAD_ROWS(BVML_ACT_TANH)
        BVML_GRAD_ROWS(BVML_ACT_SILU)
        BVML_GRAD_ROWS(BVML_ACT_GELU)
#undef BVML_GRAD_ROWS
        default: break;
    }
}

template <typename T>
__global__ void __launch_bounds__(kCols)
gated_backward_kernel(const GatedBackwardLaunch L, bool vec_h, bool vec_g, bool vec_u, bool vec_d) {
    const int lane = threadIdx.x % 32, ry = threadIdx.x / 32;
    const int c = blockIdx.x * kCols + lane * 8;
    if (c >= L.F) return;
    // two rows at a time: six loads in flight a thread
    const long long stride = (long long)gridDim.y * kRowThreads;
    for (long long t0 = (long long)blockIdx.y * kRowThreads + ry; t0 < L.T; t0 += 2 * stride) {
        float dh[2][8], g[2][8], u[2][8];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const long long t = t0 + i * stride < L.T ? t0 + i * stride : t0;
            load_cols(static_cast<const T*>(L.dh) + t * L.lddh, c, L.F, vec_h, dh[i]);
            load_cols(static_cast<const T*>(L.g) + t * L.ldg, c, L.F, vec_g, g[i]);
            load_cols(static_cast<const T*>(L.u) + t * L.ldu, c, L.F, vec_u, u[i]);
        }
        grad_rows(L.act, dh, g, u);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const long long t = t0 + i * stride;
            if (t >= L.T) continue;
            store_cols(static_cast<T*>(L.dg) + t * L.ldd, c, L.F, vec_d, g[i]);
            store_cols(static_cast<T*>(L.du) + t * L.ldd, c, L.F, vec_d, u[i]);
        }
    }
}

int row_blocks(int T, int N) {
    const long long cols = ((long long)N + kCols - 1) / kCols;
    const long long rows = ((long long)T + kRowThreads - 1) / kRowThreads;
    // about eight blocks an SM (148) in all: enough bytes in flight, few partial sums
    long long want = (148 * 8 + cols - 1) / cols;
    return (int)(want < rows ? want : rows);
}

}  // namespace

int act_backward_parts(int T, int N) { return row_blocks(T, N); }

cudaError_t launch_act_backward(const ActBackwardLaunch& L, cudaStream_t s) {
    if (L.T == 0) return cudaSuccess;
    const dim3 grid((L.N + kCols - 1) / kCols, row_blocks(L.T, L.N));
    const bool a = on16(L.dy, L.lddy, 2), b = L.z && on16(L.z, L.ldz, 2),
               c = L.dz && on16(L.dz, L.lddz, 2);
    if (L.type == BVML_F16) act_backward_kernel<__half><<<grid, kCols, 0, s>>>(L, a, b, c);
    else act_backward_kernel<__nv_bfloat16><<<grid, kCols, 0, s>>>(L, a, b, c);
    return cudaGetLastError();
}

cudaError_t launch_gated_backward(const GatedBackwardLaunch& L, cudaStream_t s) {
    if (L.T == 0) return cudaSuccess;
    const dim3 grid((L.F + kCols - 1) / kCols, row_blocks(L.T, L.F));
    const bool a = on16(L.dh, L.lddh, 2), b = on16(L.g, L.ldg, 2), c = on16(L.u, L.ldu, 2),
               d = on16(L.dg, L.ldd, 2) && on16(L.du, L.ldd, 2);
    if (L.type == BVML_F16) gated_backward_kernel<__half><<<grid, kCols, 0, s>>>(L, a, b, c, d);
    else gated_backward_kernel<__nv_bfloat16><<<grid, kCols, 0, s>>>(L, a, b, c, d);
    return cudaGetLastError();
}

}  // namespace blocks
}  // namespace bvml
