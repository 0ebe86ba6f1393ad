// Shared by the feed-forward operators' kernels (libbvml_blocks.so, sm_100a):
// element types, activations and their derivatives, 16-byte vector access.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../bvml_common.cuh"
#include "bvml_blocks.h"

#if defined(__CUDA_ARCH__) && (__CUDA_ARCH__ < 1000)
#error "brovisionml_b200 kernels are written for sm_100a (B200) only"
#endif

namespace bvml {
namespace blocks {

// Every kernel here is launched as a programmatic dependent of the one before it
// in the stream (launch_pdl): it may be resident before that one has ended, so each
// calls begin() before it touches global memory, once what its CTA holds on to
// (TMEM) has been allocated; the next kernel may come then. Loads are ordinary ones:
// what the kernel before wrote is not read-only for this one's whole life, as
// __ldg and __restrict__ would have it.
__device__ __forceinline__ void begin() {
    pdl_trigger();
    pdl_wait();
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// Two values as a pair of 16-bit elements, in one (packed) conversion: single ones
// run at a quarter of the rate.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(h);
}

// Eight consecutive elements as floats; p on 16 bytes.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(p);
        const float4 b = *reinterpret_cast<const float4*>(p + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f(e[i]);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]),
                                                  pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
}

// The hardware's 2^x and 1 / x, results below 2^-126 flushed to zero: the instructions that
// subnormal results would take bound the elementwise kernels. What is added to 1 next loses
// nothing by it; sigmoid and exp(-z^2 / 2) are zero where they would be smaller, and so
// silu for z below -87.3 and gelu below -13.1, both within |z| 2^-126 of their values, which
// bf16 and fp32 could still hold.
__device__ __forceinline__ float ex2(float x) {
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x));
    return x;
}
__device__ __forceinline__ float rcp(float x) {
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x));
    return x;
}
constexpr float kLog2E = 1.4426950408889634f;
// sigmoid: exp overflows to infinity for z below -88, where 1 / inf = 0 is the
// value. A relative error of a few 2^-24 and |z| 2^-24, on what is rounded to 16
// bits as a rule.
__device__ __forceinline__ float sigmoid_f(float z) { return rcp(1.0f + ex2(-kLog2E * z)); }

constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;

// The normal distribution function, and e = exp(-z^2 / 2) on the way, without a
// branch (erff takes two paths, which lanes and unrolled elements walk one
// after the other: 50 us on an 8192 x 8192 epilogue). With x = |z| / sqrt 2 and
// t = 1 / (1 + 0.3 x), Phi(-|z|) = exp(-x^2) erfc(x) exp(x^2) / 2, and erfc(x) exp(x^2) / t
// is smooth in t on (0, 1]: a polynomial of degree 8, fitted here for the least relative
// error (3.1e-8 in exact arithmetic, as far as exp(-z^2 / 2) is not zero; in fp32 6e-7 of
// Phi for |z| < 4).
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    const float t = rcp(fmaf(0.3f * kSqrtHalf, fabsf(z), 1.0f));
    e = ex2(-0.5f * kLog2E * z * z);
    float q = -0.12952278554439545f;
    q = fmaf(q, t, 0.48556262254714966f);
    q = fmaf(q, t, -0.5122768878936768f);
    q = fmaf(q, t, 0.5477187037467957f);
    q = fmaf(q, t, -0.09464981406927109f);
    q = fmaf(q, t, 0.21492567658424377f);
    q = fmaf(q, t, 0.14833925664424896f);
    q = fmaf(q, t, 0.17071521282196045f);
    q = fmaf(q, t, 0.1691880077123642f);
    q *= 0.5f * e * t;
    return z < 0.0f ? q : 1.0f - q;
}

// The activations of bvml_blocks.h. NaN stays NaN (relu compares, it does not
// take a maximum, which would drop it).
__device__ __forceinline__ float act_f(float z, int act) {
    switch (act) {
        case BVML_ACT_RELU: return z < 0.0f ? 0.0f : z;
        case BVML_ACT_SIGMOID: return sigmoid_f(z);
        case BVML_ACT_TANH: return tanhf(z);
        case BVML_ACT_SILU: return z * sigmoid_f(z);
        case BVML_ACT_GELU: { float e; return z * normal_cdf(z, e); }
        default: return z;
    }
}

// Sigmoid's and tanh's derivatives: c a / (1 + a)^2 with a = 2^(k |z|), that is exp(-|z|)
// and c = 1 or exp(-2 |z|) and c = 4. f (1 - f) and 1 - f^2 cancel, at z = 8 down to a
// seventh of tanh's value. Relative error below (4 |z| + 16) 2^-24.
__device__ __forceinline__ float bell_f(float z, float k, float c) {
    const float a = ex2(k * fabsf(z)), r = rcp(1.0f + a);
    return a * r * (c * r);
}

// ... and their derivatives: value and derivative share what they can.
__device__ __forceinline__ void act_grad_f(float z, int act, float& f, float& d) {
    switch (act) {
        case BVML_ACT_RELU:
            f = z < 0.0f ? 0.0f : z;
            d = z > 0.0f ? 1.0f : 0.0f;
            break;
        case BVML_ACT_SIGMOID: {
            f = sigmoid_f(z);
            d = bell_f(z, -kLog2E, 1.0f);
            break;
        }
        case BVML_ACT_TANH: {
            f = tanhf(z);
            d = bell_f(z, -2.0f * kLog2E, 4.0f);
            break;
        }
        case BVML_ACT_SILU: {
            const float p = sigmoid_f(z);
            f = z * p;
            d = p * (1.0f + z * (1.0f - p));
            break;
        }
        case BVML_ACT_GELU: {
            float e;
            const float phi = normal_cdf(z, e);
            f = z * phi;
            d = fmaf(z * kInvSqrt2Pi, e, phi);
            break;
        }
        default: f = z; d = 1.0f;
    }
}

}  // namespace blocks
}  // namespace bvml
