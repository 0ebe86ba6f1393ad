// Shared by the feed-forward operators' kernels (libbvml_blocks.so, sm_100a):
// element types, activations and their derivatives, 16-byte vector access.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "bvml_blocks.h"

#if defined(__CUDA_ARCH__) && (__CUDA_ARCH__ < 1000)
#error "brovisionml_b200 kernels are written for sm_100a (B200) only"
#endif

namespace bvml {
namespace blocks {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
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
        uint4 u;
        T* e = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_f<T>(v[i]);
        *reinterpret_cast<uint4*>(p) = u;
    }
}

// sigmoid: exp overflows to infinity for z below -88, where 1 / inf = 0 is the
// value. The fast exponential and division: a relative error of a few 2^-24 and
// |z| 2^-24 (on what is rounded to 16 bits as a rule), in a third of the
// instructions, which bound the elementwise kernels.
__device__ __forceinline__ float sigmoid_f(float z) {
    return __fdividef(1.0f, 1.0f + __expf(-z));
}

constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;

// The activations of bvml_blocks.h. NaN stays NaN (relu compares, it does not
// take a maximum, which would drop it).
__device__ __forceinline__ float act_f(float z, int act) {
    switch (act) {
        case BVML_ACT_RELU: return z < 0.0f ? 0.0f : z;
        case BVML_ACT_SIGMOID: return sigmoid_f(z);
        case BVML_ACT_TANH: return tanhf(z);
        case BVML_ACT_SILU: return z * sigmoid_f(z);
        case BVML_ACT_GELU: return 0.5f * z * (1.0f + erff(z * kSqrtHalf));
        default: return z;
    }
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
            d = f * (1.0f - f);
            break;
        }
        case BVML_ACT_TANH: {
            f = tanhf(z);
            d = 1.0f - f * f;
            break;
        }
        case BVML_ACT_SILU: {
            const float p = sigmoid_f(z);
            f = z * p;
            d = p * (1.0f + z * (1.0f - p));
            break;
        }
        case BVML_ACT_GELU: {
            const float phi = 0.5f * (1.0f + erff(z * kSqrtHalf));
            f = z * phi;
            d = phi + z * kInvSqrt2Pi * __expf(-0.5f * z * z);
            break;
        }
        default: f = z; d = 1.0f;
    }
}

}  // namespace blocks
}  // namespace bvml
