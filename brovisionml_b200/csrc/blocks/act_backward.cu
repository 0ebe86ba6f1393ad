// The elementwise half of the products' backward passes:
//   linear  dz = dy act'(z), and the bias gradient's sums over rows of dz
//   gated   dg = dh u act'(g), du = dh act(g)
//
// Each input is read once, 16 bytes a thread and access; a block covers up to
// 2048 columns and walks rows, the next rows' loads in flight; a thread keeps eight
// columns' sums in registers. The sums over a block's rows and over blocks run in
// a fixed order. What the matrix products read back (dz, dg, du) is rounded to 16
// bits, the type the tensor cores take, which makes the gradients' error against 64 bits 1.41
// times that of one rounding at the end (fp16 2.1e-4 -> 2.9e-4 of their size, bf16 1.7e-3 ->
// 2.3e-3); what the rounding leaves over, as a second operand, would double the products.
// The bias gradient sums the 32-bit values.
//
// Bound by HBM where the rows are many (gated, 8191 x 5632: 80 us, 5.8 TB/s), by
// issuing (26 instructions an element) where L2 holds them (4099 x 2056 fp16: 14 us).
#include "blocks_common.cuh"
#include "blocks_internal.h"

namespace bvml {
namespace blocks {
namespace {

constexpr int kThreads = 256;

// Up to eight columns c .. of row pointer p; what lies past n is left.
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

// Eight columns as stored, asked for ahead of use.
template <typename T>
struct alignas(16) Raw {
    T e[8];
};
template <typename T>
__device__ __forceinline__ void ask_cols(const T* p, int c, int n, bool vec, Raw<T>& r) {
    if (vec && c + 8 <= n) {
        *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p + c);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) r.e[e] = c + e < n ? p[c + e] : from_f<T>(0.0f);
    }
}

// v <- v act'(z); the activation is chosen outside the loop
__device__ __forceinline__ void times_grad(int act, const float (&z)[8], float (&v)[8]) {
    switch (act) {
#define BVML_TIMES_GRAD(code)                             \
    case code:                                            \
        _Pragma("unroll") for (int e = 0; e < 8; ++e) {   \
            float f, d;                                   \
            act_grad_f(z[e], code, f, d);                 \
            v[e] *= d;                                    \
        }                                                 \
        break;
        // one path for these two: with one each the kernel spills (12 bytes loaded -> 36)
        case BVML_ACT_SIGMOID:
        case BVML_ACT_TANH: {
            const float k = act == BVML_ACT_TANH ? -2.0f * kLog2E : -kLog2E;
            const float c = act == BVML_ACT_TANH ? 4.0f : 1.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= bell_f(z[e], k, c);
            break;
        }
        BVML_TIMES_GRAD(BVML_ACT_RELU)
        BVML_TIMES_GRAD(BVML_ACT_SILU)
        BVML_TIMES_GRAD(BVML_ACT_GELU)
#undef BVML_TIMES_GRAD
        default: break;
    }
}

// A block covers `span` threads of eight columns by blockDim.x / span rows at a time.
template <typename T>
__global__ void __launch_bounds__(kThreads, 4)
act_backward_kernel(const ActBackwardLaunch L, int span, bool vec_dy, bool vec_z, bool vec_dz) {
    __shared__ float sh[kThreads * 8];
    const int x = threadIdx.x % span, ry = threadIdx.x / span, rows = blockDim.x / span;
    const int c = (blockIdx.x * span + x) * 8;
    begin();
    float sum[8] = {};
    const long long stride = (long long)gridDim.y * rows;
    if (c < L.N) {
        // the next two rows' loads are in flight while a row is computed
        Raw<T> rd[2], rz[2];
        auto ask = [&](long long t, int i) {
            if (t >= L.T) return;
            ask_cols(static_cast<const T*>(L.dy) + t * L.lddy, c, L.N, vec_dy, rd[i]);
            if (L.z) ask_cols(static_cast<const T*>(L.z) + t * L.ldz, c, L.N, vec_z, rz[i]);
        };
        const long long t0 = (long long)blockIdx.y * rows + ry;
        ask(t0, 0);
        ask(t0 + stride, 1);
        for (long long t = t0; t < L.T;) {
#pragma unroll
            for (int i = 0; i < 2; ++i, t += stride) {
                if (t >= L.T) break;
                float d[8], z[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    d[e] = to_f(rd[i].e[e]);
                    z[e] = to_f(rz[i].e[e]);
                }
                ask(t + 2 * stride, i);
                if (L.z) times_grad(L.act, z, d);
                if (L.dz) store_cols(static_cast<T*>(L.dz) + t * L.lddz, c, L.N, vec_dz, d);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] += d[e];
            }
        }
    }
    if (!L.partial) return;
    // the block's rows side by side, added in their order
#pragma unroll
    for (int e = 0; e < 8; ++e) sh[threadIdx.x * 8 + e] = sum[e];
    __syncthreads();
    for (int i = threadIdx.x; i < span * 8; i += blockDim.x) {
        const int n = blockIdx.x * span * 8 + i;
        if (n >= L.N) break;
        float v = sh[i];
        for (int r = 1; r < rows; ++r) v += sh[r * span * 8 + i];
        L.partial[(long long)blockIdx.y * L.N + n] = v;
    }
}

// g, u <- dh u act'(g), dh act(g); the activation is chosen outside the loop
__device__ __forceinline__ void grad_cols(int act, const float (&dh)[8], float (&g)[8],
                                          float (&u)[8]) {
    switch (act) {
#define BVML_GRAD_COLS(code)                              \
    case code:                                            \
        _Pragma("unroll") for (int e = 0; e < 8; ++e) {   \
            float f, d;                                   \
            act_grad_f(g[e], code, f, d);                 \
            g[e] = dh[e] * u[e] * d;                      \
            u[e] = dh[e] * f;                             \
        }                                                 \
        break;
        BVML_GRAD_COLS(BVML_ACT_RELU)
        BVML_GRAD_COLS(BVML_ACT_SIGMOID)
        BVML_GRAD_COLS(BVML_ACT_TANH)
        BVML_GRAD_COLS(BVML_ACT_SILU)
        BVML_GRAD_COLS(BVML_ACT_GELU)
#undef BVML_GRAD_COLS
        default: break;
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4)
gated_backward_kernel(const GatedBackwardLaunch L, int span, bool vec_h, bool vec_g, bool vec_u,
                      bool vec_d) {
    const int x = threadIdx.x % span, ry = threadIdx.x / span, rows = blockDim.x / span;
    const int c = (blockIdx.x * span + x) * 8;
    begin();
    if (c >= L.F) return;
    const long long stride = (long long)gridDim.y * rows;
    // the next row's loads are in flight while this one is computed
    Raw<T> rh, rg, ru;
    auto ask = [&](long long t) {
        if (t >= L.T) return;
        ask_cols(static_cast<const T*>(L.dh) + t * L.lddh, c, L.F, vec_h, rh);
        ask_cols(static_cast<const T*>(L.g) + t * L.ldg, c, L.F, vec_g, rg);
        ask_cols(static_cast<const T*>(L.u) + t * L.ldu, c, L.F, vec_u, ru);
    };
    ask((long long)blockIdx.y * rows + ry);
    for (long long t = (long long)blockIdx.y * rows + ry; t < L.T; t += stride) {
        float dh[8], g[8], u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            dh[e] = to_f(rh.e[e]);
            g[e] = to_f(rg.e[e]);
            u[e] = to_f(ru.e[e]);
        }
        ask(t + stride);
        grad_cols(L.act, dh, g, u);
        store_cols(static_cast<T*>(L.dg) + t * L.ldd, c, L.F, vec_d, g);
        store_cols(static_cast<T*>(L.du) + t * L.ldd, c, L.F, vec_d, u);
    }
}

// How a row of N is covered: `blocks` blocks of `span` threads, eight columns each,
// evenly (a row of 2056 is 2 x 129 threads and not 256 and one), `rows` rows a block.
struct Cover {
    int span, rows, blocks;
};
Cover cover(int N) {
    const int units = (int)(((long long)N + 7) / 8);
    Cover c;
    c.blocks = (units + kThreads - 1) / kThreads;
    c.span = (units + c.blocks - 1) / c.blocks;
    c.rows = kThreads / c.span;
    return c;
}
// Blocks along the rows: 1024 threads an SM (148) in all, what is resident at
// once, so that there are bytes enough in flight and few partial sums.
// `turns` times as many where nothing is summed: blocks that start as others end
// keep the loads coming (gated, 8191 x 5632: 80 us with two turns, 92 with one).
int row_blocks(int T, int N, int turns) {
    const Cover c = cover(N);
    const long long rows = ((long long)T + c.rows - 1) / c.rows;
    const int per_sm = 1024 / ((c.span * c.rows + 31) / 32 * 32);
    const long long want = (148LL * per_sm * turns + c.blocks - 1) / c.blocks;
    return (int)(want < rows ? want : rows);
}

}  // namespace

int act_backward_parts(int T, int N) { return row_blocks(T, N, 1); }

cudaError_t launch_act_backward(const ActBackwardLaunch& L, cudaStream_t s) {
    if (L.T == 0) return cudaSuccess;
    const Cover v = cover(L.N);
    const dim3 grid(v.blocks, row_blocks(L.T, L.N, 1));
    const int span = v.span, threads = v.span * v.rows;
    const bool a = on16(L.dy, L.lddy, 2), b = L.z && on16(L.z, L.ldz, 2),
               c = L.dz && on16(L.dz, L.lddz, 2);
    if (L.type == BVML_F16)
        return launch_pdl(act_backward_kernel<__half>, grid, threads, 0, s, true, L, span, a, b, c);
    return launch_pdl(act_backward_kernel<__nv_bfloat16>, grid, threads, 0, s, true, L, span, a, b, c);
}

cudaError_t launch_gated_backward(const GatedBackwardLaunch& L, cudaStream_t s) {
    if (L.T == 0) return cudaSuccess;
    const Cover v = cover(L.F);
    const dim3 grid(v.blocks, row_blocks(L.T, L.F, 2));
    const int span = v.span, threads = v.span * v.rows;
    const bool a = on16(L.dh, L.lddh, 2), b = on16(L.g, L.ldg, 2), c = on16(L.u, L.ldu, 2),
               d = on16(L.dg, L.ldd, 2) && on16(L.du, L.ldd, 2);
    if (L.type == BVML_F16)
        return launch_pdl(gated_backward_kernel<__half>, grid, threads, 0, s, true, L, span, a, b, c, d);
    return launch_pdl(gated_backward_kernel<__nv_bfloat16>, grid, threads, 0, s, true, L, span, a, b, c, d);
}

}  // namespace blocks
}  // namespace bvml
