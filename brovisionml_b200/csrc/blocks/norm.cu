// RMS norm over rows of K features, with the residual's addition before it,
// a 16 / 32-bit or an 8-bit output, and its backward pass.
//
//   forward   s = x + r,  q = sum_k s^2,  y = s * rsqrt(q / K + eps) * w
//   8 bits    max_k |y| = rstd * max_k |s w|, so the row's scale comes out of
//             the same reduction as q: one pass over the row
//   backward  n = s rstd:  dx = rstd (dy w - n mean(dy w n)) + ds, dw = sum_t dy n
//
// Bound by HBM: every row is read once into registers (G threads a row, VPT
// groups of eight elements a thread), reduced, and written from there. Rows of
// up to 512 features belong to a warp or part of one (no block barrier), longer
// ones to a block; beyond 16 Ki features a block walks the row twice, the second
// time out of L2, an element a thread and load. A block keeps its weights in registers
// over its rows, and the backward pass its sums of dw, which it writes once: the sums
// over blocks are a second small kernel, in a fixed order (no atomics).
//
// us (TB/s): 57600 x 128 fp16 6.6 (4.5; 6.85 with sums of squares and of the residual
// element by element and not in pairs), 8197 x 4096 bf16 with residual to 8 bits 40 to
// 44 (5.3 to 5.9; in pairs its quotients took 2 us longer), backward 16384 x 2048 bf16
// 52.9 (5.1, the second kernel included); one row of 4096 5.0, the launch. By width, bf16,
// T K = 33.5 M, forward and backward: 4096 25.7 (5.2) and 41.7 (4.8), 8192 29.4 and 42.8,
// 12000 27.4 and 125 (four groups a thread do not fit the registers: 536 bytes spilled),
// 16384 24.7 and 101, 16392 60.9 (2.2) and 157 (1.3), 20000 77.9 and 161.
#include "blocks_common.cuh"
#include "blocks_internal.h"

namespace bvml {
namespace blocks {
namespace {

constexpr int kNormThreads = 256;  // rows of at most a warp share a block of this size
constexpr int kLongThreads = 512;
// Below this a row's largest |y| counts as zero (its scale would come near the smallest
// normal numbers).
constexpr float kTinyMax = 0x1p-110f;
// Rows whose largest |s w| is below kSmallMax are lifted by a power of two on their way to
// 8 bits: 448 / max |s w| would overflow.
constexpr float kSmallMax = 0x1p-100f, kLift = 0x1p60f;
__device__ __forceinline__ float lift_of(float m) { return m < kSmallMax ? kLift : 1.0f; }

struct NormArgs {
    const void *x, *r, *w;
    void *y, *sum;
    float* scale;
    long long ldx, ldr, ldy, lds;
    int T, K;
    int w32;  // weights are fp32 (else the rows' type)
    int vec;  // every row starts on 16 bytes and K is a multiple of 8
    float eps;
};

struct NormBwdArgs {
    const void *dy, *s, *w, *ds;
    void* dx;
    float* partial;
    long long lddy, lds, ldds, lddx;
    int T, K, w32, vec;
    float eps;
};

// From a row's largest |s w| to its scale and to y / scale = s w 448 / max |s w|,
// from which the root drops out. What the products and the quotient leave over in
// 32 bits is carried along (`rest` of the largest, `lo` of the quotient): a value
// next to a rounding border of the 8 bits then falls where the formula has it, but
// for the one rounding to 32 bits before the one to 8. s: the row's, times lift_of(m).
struct Quant {
    float scale, hi, lo;
    __device__ __forceinline__ float operator()(float s, float w) const {
        const float p = s * w, rest = fmaf(s, w, -p);
        return fmaf(p, hi, fmaf(p, lo, rest * hi));
    }
};
__device__ __forceinline__ Quant quant_of(float m, float rest, float rstd) {
    const float top = m * rstd;
    if (top < kTinyMax) return Quant{1.0f, 0.0f, 0.0f};
    Quant f;
    f.scale = top / 448.0f;
    const float most = m * lift_of(m);
    f.hi = 448.0f / most;
    f.lo = (fmaf(-most, f.hi, 448.0f) - rest * lift_of(m) * f.hi) / most;
    // NaN or an infinity in the row (1 / infinity is zero), or |s w| past the largest number
    if (!(top <= 3.4028235e38f)) f.scale = f.hi = __int_as_float(0x7fffffff);
    return f;
}
// The larger of two, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(a), "f"(b));
    return a;
}
// A thread's largest |s w| as its product rounded to 32 bits, m, and what that left over,
// the larger of two where the rounded products are equal: every thread of a row, in whatever
// order, must arrive at the same pair. Rounding keeps the products' order, so that rest is
// the largest of |s w| - m, exact for m's own product. Each group of eight on its own,
// then joined, as chains of maxima are what a row waits for. m: NaN stays.
template <int VPT>
__device__ __forceinline__ void largest(const float (&s)[VPT][8], const float (&w)[VPT][8],
                                        float& m, float& rest) {
    float g[VPT][2], r[VPT][2];
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            g[v][h] = fabsf(s[v][h] * w[v][h]);
#pragma unroll
            for (int e = 2 + h; e < 8; e += 2) g[v][h] = max_nan(g[v][h], fabsf(s[v][e] * w[v][e]));
        }
    m = max_nan(g[0][0], g[0][1]);
#pragma unroll
    for (int v = 1; v < VPT; ++v) m = max_nan(m, max_nan(g[v][0], g[v][1]));
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            r[v][h] = fmaf(fabsf(s[v][h]), fabsf(w[v][h]), -m);
#pragma unroll
            for (int e = 2 + h; e < 8; e += 2)
                r[v][h] = fmaxf(r[v][h], fmaf(fabsf(s[v][e]), fabsf(w[v][e]), -m));
        }
    rest = fmaxf(r[0][0], r[0][1]);
#pragma unroll
    for (int v = 1; v < VPT; ++v) rest = fmaxf(rest, fmaxf(r[v][0], r[v][1]));
}

// Feature index of element e of group v of lane l: eight consecutive features
// where vectors can be used, otherwise lanes side by side.
template <int G>
__device__ __forceinline__ int feature(int vec, int v, int e, int l) {
    return vec ? (v * G + l) * 8 + e : (v * 8 + e) * G + l;
}

template <typename T, int G, int VPT>
__device__ __forceinline__ void load_row(const T* p, int K, int vec, int l, float (&o)[VPT][8]) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        if (vec) {
            const int k = (v * G + l) * 8;
            if (k < K) {
                load8(p + k, o[v]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) o[v][e] = 0.0f;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int k = (v * 8 + e) * G + l;
                o[v][e] = k < K ? to_f(p[k]) : 0.0f;
            }
        }
    }
}

// Eight elements as stored: what a thread keeps of a row that it has asked for
// and not used yet.
template <typename T>
struct alignas(16) Raw {
    T e[8];
};
template <typename T, int G, int VPT>
__device__ __forceinline__ void fetch_row(const T* p, int K, int vec, int l, Raw<T> (&o)[VPT]) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        if (vec) {
            const int k = (v * G + l) * 8;
            uint4* d = reinterpret_cast<uint4*>(&o[v]);
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                d[i] = k < K ? reinterpret_cast<const uint4*>(p + k)[i] : make_uint4(0, 0, 0, 0);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int k = (v * 8 + e) * G + l;
                o[v].e[e] = k < K ? p[k] : from_f<T>(0.0f);
            }
        }
    }
}
template <typename T, int VPT>
__device__ __forceinline__ void widen(const Raw<T> (&r)[VPT], float (&o)[VPT][8]) {
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) o[v][e] = to_f(r[v].e[e]);
}

template <typename T, int G, int VPT>
__device__ __forceinline__ void store_row(T* p, int K, int vec, int l, const float (&o)[VPT][8]) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        if (vec) {
            const int k = (v * G + l) * 8;
            if (k < K) store8(p + k, o[v]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int k = (v * 8 + e) * G + l;
                if (k < K) p[k] = from_f<T>(o[v][e]);
            }
        }
    }
}

__device__ __forceinline__ uint8_t to_e4m3(float v) {
    return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

template <int G, int VPT>
__device__ __forceinline__ void store_row_e4m3(uint8_t* p, int K, int vec, int l,
                                               const float (&o)[VPT][8]) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        if (vec) {
            const int k = (v * G + l) * 8;
            if (k < K) {
                uint2 u;
                uint16_t* h = reinterpret_cast<uint16_t*>(&u);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    h[e] = __nv_cvt_float2_to_fp8x2(make_float2(o[v][2 * e], o[v][2 * e + 1]),
                                                    __NV_SATFINITE, __NV_E4M3);
                *reinterpret_cast<uint2*>(p + k) = u;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int k = (v * 8 + e) * G + l;
                if (k < K) p[k] = to_e4m3(o[v][e]);
            }
        }
    }
}

// Sum of a over the G threads of a row, and of b; every thread gets the result. G > 32: the
// whole block takes part; `slot` alternates between rows, so that one barrier a row is
// enough.
template <int G>
__device__ __forceinline__ void row_reduce(float& a, float& b, float (*slots)[3][16], int slot) {
    constexpr int kWidth = G < 32 ? G : 32;
#pragma unroll
    for (int d = kWidth / 2; d > 0; d >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, d);
        b += __shfl_xor_sync(0xffffffffu, b, d);
    }
    if constexpr (G > 32) {
        constexpr int kN = G / 32;
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0) {
            slots[slot][0][warp] = a;
            slots[slot][1][warp] = b;
        }
        __syncthreads();
        a = slots[slot][0][0];
        b = slots[slot][1][0];
#pragma unroll
        for (int i = 1; i < kN; ++i) {
            a += slots[slot][0][i];
            b += slots[slot][1][i];
        }
    }
}
// ... and the largest m (not negative; NaN if one is) with the largest c beside it.
__device__ __forceinline__ float warp_max_nan(float v) {
    asm volatile("redux.sync.max.NaN.f32 %0, %0, 0xffffffff;" : "+f"(v));
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
    asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(v));
    return v;
}
template <int G>
__device__ __forceinline__ void row_reduce_max(float& a, float& m, float& c, float (*slots)[3][16],
                                               int slot) {
    constexpr int kWidth = G < 32 ? G : 32;
#pragma unroll
    for (int d = kWidth / 2; d > 0; d >>= 1) a += __shfl_xor_sync(0xffffffffu, a, d);
    float most = m;
    if constexpr (G < 32) {
#pragma unroll
        for (int d = kWidth / 2; d > 0; d >>= 1)
            most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, d));
        c = m == most ? c : -INFINITY;
#pragma unroll
        for (int d = kWidth / 2; d > 0; d >>= 1)
            c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, d));
    } else {
        most = warp_max_nan(m);
        c = warp_max(m == most ? c : -INFINITY);
    }
    m = most;
    if constexpr (G > 32) {
        constexpr int kN = G / 32;
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0) {
            slots[slot][0][warp] = a;
            slots[slot][1][warp] = m;
            slots[slot][2][warp] = c;
        }
        __syncthreads();
        a = slots[slot][0][0];
        m = slots[slot][1][0];
#pragma unroll
        for (int i = 1; i < kN; ++i) {
            a += slots[slot][0][i];
            m = max_nan(m, slots[slot][1][i]);
        }
        c = -INFINITY;
#pragma unroll
        for (int i = 0; i < kN; ++i)
            c = fmaxf(c, slots[slot][1][i] == m ? slots[slot][2][i] : -INFINITY);
    }
}

// Blocks an SM that the forward pass is built for: 64 registers a thread with one
// group of eight, 80 with two, 128 with four.
constexpr int forward_blocks(int G, int VPT) {
    const int threads = G > 32 ? G : kNormThreads;
    const int n = (VPT == 1 ? 1024 : VPT == 2 ? 768 : 512) / threads;
    return n > 0 ? n : 1;
}

template <typename T, int G, int VPT, bool Q>
__global__ void __launch_bounds__(G > 32 ? G : kNormThreads, forward_blocks(G, VPT))
rms_norm_kernel(const NormArgs a) {
    constexpr int kThreads = G > 32 ? G : kNormThreads;
    constexpr int kRows = kThreads / G;
    __shared__ float slots[2][3][16];
    const int l = threadIdx.x % G, g = threadIdx.x / G;
    begin();
    float w[VPT][8];
    if (a.w32) load_row<float, G, VPT>(static_cast<const float*>(a.w), a.K, a.vec, l, w);
    else load_row<T, G, VPT>(static_cast<const T*>(a.w), a.K, a.vec, l, w);
    const float inv_k = 1.0f / (float)a.K;
    int slot = 0;
    // The next turn's rows are asked for before this turn's reduction, so that a
    // block has loads in flight all the time. Every thread of the block makes the
    // same number of turns (barriers, shuffles).
    const long long stride = (long long)gridDim.x * kRows;
    Raw<T> xn[VPT], rn[VPT];
    auto ask = [&](long long t) {
        if (t >= a.T) return;
        fetch_row<T, G, VPT>(static_cast<const T*>(a.x) + t * a.ldx, a.K, a.vec, l, xn);
        if (a.r)
            fetch_row<T, G, VPT>(static_cast<const T*>(a.r) + t * a.ldr, a.K, a.vec, l, rn);
    };
    ask((long long)blockIdx.x * kRows + g);
    for (long long t0 = (long long)blockIdx.x * kRows; t0 < a.T; t0 += stride, slot ^= 1) {
        const long long t = t0 + g;
        const bool in = t < a.T;
        float s[VPT][8];
        if (in) {
            widen(xn, s);
            if (a.r) {
                float r[VPT][8];
                widen(rn, r);
#pragma unroll
                for (int v = 0; v < VPT; ++v)
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const float2 d = __fadd2_rn(make_float2(s[v][e], s[v][e + 1]),
                                                    make_float2(r[v][e], r[v][e + 1]));
                        s[v][e] = d.x, s[v][e + 1] = d.y;
                    }
            }
            ask(t + stride);
            if (a.sum) store_row<T, G, VPT>(static_cast<T*>(a.sum) + t * a.lds, a.K, a.vec, l, s);
        } else {
#pragma unroll
            for (int v = 0; v < VPT; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[v][e] = 0.0f;
        }
        float2 q2 = make_float2(0.0f, 0.0f);
        float m = 0.0f, rest = 0.0f;
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float2 d = make_float2(s[v][e], s[v][e + 1]);
                q2 = __ffma2_rn(d, d, q2);
            }
        }
        if constexpr (Q) largest<VPT>(s, w, m, rest);
        float q = q2.x + q2.y;
        if constexpr (Q) row_reduce_max<G>(q, m, rest, slots, slot);
        else row_reduce<G>(q, m, slots, slot);
        if (!in) continue;
        const float rstd = rsqrtf(fmaf(q, inv_k, a.eps));
        if constexpr (Q) {
            const Quant f = quant_of(m, rest, rstd);
            if (l == 0) a.scale[t] = f.scale;
            if (m < kSmallMax) {
#pragma unroll
                for (int v = 0; v < VPT; ++v)
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[v][e] *= kLift;
            }
#pragma unroll
            for (int v = 0; v < VPT; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[v][e] = f(s[v][e], w[v][e]);
            store_row_e4m3<G, VPT>(static_cast<uint8_t*>(a.y) + t * a.ldy, a.K, a.vec, l, s);
        } else {
#pragma unroll
            for (int v = 0; v < VPT; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[v][e] *= w[v][e] * rstd;
            store_row<T, G, VPT>(static_cast<T*>(a.y) + t * a.ldy, a.K, a.vec, l, s);
        }
    }
}

// Rows of more than 16 Ki features: a block a row, two walks over it.
template <typename T, bool Q>
__global__ void __launch_bounds__(kLongThreads)
rms_norm_long_kernel(const NormArgs a) {
    __shared__ float slots[2][3][16];
    begin();
    const float inv_k = 1.0f / (float)a.K;
    int slot = 0;
    auto wt = [&](int k) {
        return a.w32 ? static_cast<const float*>(a.w)[k] : to_f(static_cast<const T*>(a.w)[k]);
    };
    for (long long t = blockIdx.x; t < a.T; t += gridDim.x, slot ^= 1) {
        const T* x = static_cast<const T*>(a.x) + t * a.ldx;
        const T* r = a.r ? static_cast<const T*>(a.r) + t * a.ldr : nullptr;
        float q = 0.0f, m = 0.0f, rest = 0.0f;
        for (int k = threadIdx.x; k < a.K; k += kLongThreads) {
            const float s = to_f(x[k]) + (r ? to_f(r[k]) : 0.0f);
            if (a.sum) static_cast<T*>(a.sum)[t * a.lds + k] = from_f<T>(s);
            q = fmaf(s, s, q);
            if constexpr (Q) {
                const float p = fabsf(s * wt(k)), left = fmaf(fabsf(s), fabsf(wt(k)), -p);
                if (!(p < m) && !(p == m && left <= rest)) rest = left;
                m = max_nan(m, p);
            }
        }
        if constexpr (Q) row_reduce_max<kLongThreads>(q, m, rest, slots, slot);
        else row_reduce<kLongThreads>(q, m, slots, slot);
        const float rstd = rsqrtf(fmaf(q, inv_k, a.eps));
        Quant f{};
        if constexpr (Q) {
            f = quant_of(m, rest, rstd);
            if (threadIdx.x == 0) a.scale[t] = f.scale;
        }
        for (int k = threadIdx.x; k < a.K; k += kLongThreads) {
            const float s = to_f(x[k]) + (r ? to_f(r[k]) : 0.0f);
            if constexpr (Q)
                static_cast<uint8_t*>(a.y)[t * a.ldy + k] = to_e4m3(f(s * lift_of(m), wt(k)));
            else
                static_cast<T*>(a.y)[t * a.ldy + k] = from_f<T>(s * (wt(k) * rstd));
        }
    }
}

// Blocks an SM that the backward pass is built for: 64 registers a thread with
// one group of eight, twice that with two, and no more with four, which spill.
constexpr int backward_blocks(int G, int VPT) {
    const int threads = G > 32 ? G : kNormThreads;
    const int n = (VPT == 1 ? 1024 : 512) / threads;
    return n > 0 ? n : 1;
}

template <typename T, int G, int VPT>
__global__ void __launch_bounds__(G > 32 ? G : kNormThreads, backward_blocks(G, VPT))
rms_norm_backward_kernel(const NormBwdArgs a) {
    constexpr int kThreads = G > 32 ? G : kNormThreads;
    constexpr int kRows = kThreads / G;
    __shared__ float slots[2][3][16];
    __shared__ float part[kRows > 1 ? kThreads * VPT * 8 : 1];
    const int l = threadIdx.x % G, g = threadIdx.x / G;
    begin();
    float w[VPT][8], dw[VPT][8];
    if (a.w32) load_row<float, G, VPT>(static_cast<const float*>(a.w), a.K, a.vec, l, w);
    else load_row<T, G, VPT>(static_cast<const T*>(a.w), a.K, a.vec, l, w);
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[v][e] = 0.0f;
    const float inv_k = 1.0f / (float)a.K;
    int slot = 0;
    const long long stride = (long long)gridDim.x * kRows;
    Raw<T> sn[VPT], dn[VPT], en[VPT];  // the next turn's rows, as in the forward pass
    auto ask = [&](long long t) {
        if (t >= a.T) return;
        fetch_row<T, G, VPT>(static_cast<const T*>(a.s) + t * a.lds, a.K, a.vec, l, sn);
        fetch_row<T, G, VPT>(static_cast<const T*>(a.dy) + t * a.lddy, a.K, a.vec, l, dn);
    };
    ask((long long)blockIdx.x * kRows + g);
    for (long long t0 = (long long)blockIdx.x * kRows; t0 < a.T; t0 += stride, slot ^= 1) {
        const long long t = t0 + g;
        const bool in = t < a.T;
        float s[VPT][8], dy[VPT][8];
        if (in) {
            widen(sn, s);
            widen(dn, dy);
            if (a.ds)  // used after the reduction
                fetch_row<T, G, VPT>(static_cast<const T*>(a.ds) + t * a.ldds, a.K, a.vec, l, en);
            ask(t + stride);
        } else {
#pragma unroll
            for (int v = 0; v < VPT; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[v][e] = dy[v][e] = 0.0f;
        }
        float q = 0.0f, p = 0.0f;
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                q = fmaf(s[v][e], s[v][e], q);
                p = fmaf(dy[v][e] * w[v][e], s[v][e], p);
            }
        }
        row_reduce<G>(q, p, slots, slot);
        if (!in) continue;
        const float rstd = rsqrtf(fmaf(q, inv_k, a.eps));
        const float c = p * inv_k * rstd * rstd;
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                dw[v][e] = fmaf(dy[v][e], s[v][e] * rstd, dw[v][e]);
                s[v][e] = rstd * fmaf(dy[v][e], w[v][e], -s[v][e] * c);
            }
        }
        if (a.ds) {
            widen(en, dy);
#pragma unroll
            for (int v = 0; v < VPT; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[v][e] += dy[v][e];
        }
        store_row<T, G, VPT>(static_cast<T*>(a.dx) + t * a.lddx, a.K, a.vec, l, s);
    }
    float* out = a.partial + (long long)blockIdx.x * a.K;
    if constexpr (kRows > 1) {
        // the block's rows side by side: part[g][feature], summed in the order of g
        constexpr int kPer = G * VPT * 8;
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) part[g * kPer + feature<G>(a.vec, v, e, l)] = dw[v][e];
        __syncthreads();
        for (int k = threadIdx.x; k < a.K; k += kThreads) {
            float v = part[k];
#pragma unroll 4
            for (int i = 1; i < kRows; ++i) v += part[i * kPer + k];
            out[k] = v;
        }
    } else {
        store_row<float, G, VPT>(out, a.K, a.vec, l, dw);
    }
}

template <typename T>
__global__ void __launch_bounds__(kLongThreads)
rms_norm_backward_long_kernel(const NormBwdArgs a) {
    __shared__ float slots[2][3][16];
    begin();
    const float inv_k = 1.0f / (float)a.K;
    float* out = a.partial + (long long)blockIdx.x * a.K;
    auto wt = [&](int k) {
        return a.w32 ? static_cast<const float*>(a.w)[k] : to_f(static_cast<const T*>(a.w)[k]);
    };
    int slot = 0;
    bool first = true;
    for (long long t = blockIdx.x; t < a.T; t += gridDim.x, slot ^= 1) {
        const T* s = static_cast<const T*>(a.s) + t * a.lds;
        const T* dy = static_cast<const T*>(a.dy) + t * a.lddy;
        float q = 0.0f, p = 0.0f;
        for (int k = threadIdx.x; k < a.K; k += kLongThreads) {
            const float sv = to_f(s[k]);
            q = fmaf(sv, sv, q);
            p = fmaf(to_f(dy[k]) * wt(k), sv, p);
        }
        row_reduce<kLongThreads>(q, p, slots, slot);
        const float rstd = rsqrtf(fmaf(q, inv_k, a.eps));
        const float c = p * inv_k * rstd * rstd;
        for (int k = threadIdx.x; k < a.K; k += kLongThreads) {
            const float sv = to_f(s[k]), d = to_f(dy[k]);
            float o = rstd * fmaf(d, wt(k), -sv * c);
            if (a.ds) o += to_f(static_cast<const T*>(a.ds)[t * a.ldds + k]);
            static_cast<T*>(a.dx)[t * a.lddx + k] = from_f<T>(o);
            out[k] = fmaf(d, sv * rstd, first ? 0.0f : out[k]);  // a thread's own columns
        }
        first = false;
    }
}

// 16 columns a block, 32 rows side by side
template <typename T>
__global__ void __launch_bounds__(512)
column_sum_kernel(const float* part, int rows, int cols, T* out) {
    __shared__ float sh[32][17];
    const int x = threadIdx.x % 16, c = blockIdx.x * 16 + x, r0 = threadIdx.x / 16;
    begin();
    float v = 0.0f;
    if (c < cols) {
#pragma unroll 8
        for (int r = r0; r < rows; r += 32) v += part[(long long)r * cols + c];
    }
    sh[r0][x] = v;
    __syncthreads();
    if (r0 == 0 && c < cols) {
#pragma unroll
        for (int i = 1; i < 32; ++i) v += sh[i][x];
        out[c] = from_f<T>(v);
    }
}

// Threads a row and groups of eight a thread, by the row's length: the fewest
// registers that hold it.
enum class Shape { G8, G16, G32x1, G32x2, G128x1, G256x1, G256x2, G512x2, G512x4, Long };
Shape shape_of(int K) {
    if (K <= 64) return Shape::G8;
    if (K <= 128) return Shape::G16;
    if (K <= 256) return Shape::G32x1;
    if (K <= 512) return Shape::G32x2;
    if (K <= 1024) return Shape::G128x1;
    if (K <= 2048) return Shape::G256x1;
    if (K <= 4096) return Shape::G256x2;
    if (K <= 8192) return Shape::G512x2;
    if (K <= 16384) return Shape::G512x4;
    return Shape::Long;
}
int block_rows(Shape h) {
    switch (h) {
        case Shape::G8: return 32;
        case Shape::G16: return 16;
        case Shape::G32x1:
        case Shape::G32x2: return 8;
        default: return 1;
    }
}

template <typename T, bool Q>
cudaError_t norm_by_shape(Shape h, int grid, const NormArgs& a, cudaStream_t s) {
    switch (h) {
        case Shape::G8: return launch_pdl(rms_norm_kernel<T, 8, 1, Q>, grid, 256, 0, s, true, a);
        case Shape::G16: return launch_pdl(rms_norm_kernel<T, 16, 1, Q>, grid, 256, 0, s, true, a);
        case Shape::G32x1: return launch_pdl(rms_norm_kernel<T, 32, 1, Q>, grid, 256, 0, s, true, a);
        case Shape::G32x2: return launch_pdl(rms_norm_kernel<T, 32, 2, Q>, grid, 256, 0, s, true, a);
        case Shape::G128x1: return launch_pdl(rms_norm_kernel<T, 128, 1, Q>, grid, 128, 0, s, true, a);
        case Shape::G256x1: return launch_pdl(rms_norm_kernel<T, 256, 1, Q>, grid, 256, 0, s, true, a);
        case Shape::G256x2: return launch_pdl(rms_norm_kernel<T, 256, 2, Q>, grid, 256, 0, s, true, a);
        case Shape::G512x2: return launch_pdl(rms_norm_kernel<T, 512, 2, Q>, grid, 512, 0, s, true, a);
        case Shape::G512x4: return launch_pdl(rms_norm_kernel<T, 512, 4, Q>, grid, 512, 0, s, true, a);
        case Shape::Long: return launch_pdl(rms_norm_long_kernel<T, Q>, grid, kLongThreads, 0, s, true, a);
    }
    return cudaErrorInvalidValue;
}

template <typename T>
cudaError_t norm_backward_by_shape(Shape h, int grid, const NormBwdArgs& a, cudaStream_t s) {
    switch (h) {
        case Shape::G8: return launch_pdl(rms_norm_backward_kernel<T, 8, 1>, grid, 256, 0, s, true, a);
        case Shape::G16: return launch_pdl(rms_norm_backward_kernel<T, 16, 1>, grid, 256, 0, s, true, a);
        case Shape::G32x1: return launch_pdl(rms_norm_backward_kernel<T, 32, 1>, grid, 256, 0, s, true, a);
        case Shape::G32x2: return launch_pdl(rms_norm_backward_kernel<T, 32, 2>, grid, 256, 0, s, true, a);
        case Shape::G128x1: return launch_pdl(rms_norm_backward_kernel<T, 128, 1>, grid, 128, 0, s, true, a);
        case Shape::G256x1: return launch_pdl(rms_norm_backward_kernel<T, 256, 1>, grid, 256, 0, s, true, a);
        case Shape::G256x2: return launch_pdl(rms_norm_backward_kernel<T, 256, 2>, grid, 256, 0, s, true, a);
        case Shape::G512x2: return launch_pdl(rms_norm_backward_kernel<T, 512, 2>, grid, 512, 0, s, true, a);
        case Shape::G512x4: return launch_pdl(rms_norm_backward_kernel<T, 512, 4>, grid, 512, 0, s, true, a);
        case Shape::Long:
            return launch_pdl(rms_norm_backward_long_kernel<T>, grid, kLongThreads, 0, s, true, a);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t sm_count(int* sms) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    return cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
}

cudaError_t launch_rms_norm(const NormLaunch& L, cudaStream_t s) {
    if (L.T == 0) return cudaSuccess;
    int sms = 0;
    cudaError_t e = sm_count(&sms);
    if (e != cudaSuccess) return e;
    const size_t es = elem_size(L.type);
    NormArgs a{L.x, L.r, L.w, L.y, L.sum, L.scale, L.ldx, L.ldr, L.ldy, L.lds, L.T, L.K};
    a.w32 = L.wtype == BVML_F32;
    a.eps = L.eps;
    const bool y_ok = L.scale ? ((reinterpret_cast<uintptr_t>(L.y) | (uintptr_t)L.ldy) & 7) == 0
                              : on16(L.y, L.ldy, es);
    a.vec = L.K % 8 == 0 && on16(L.x, L.ldx, es) && (!L.r || on16(L.r, L.ldr, es)) &&
            on16(L.w, 0, 1) && y_ok && (!L.sum || on16(L.sum, L.lds, es));
    const Shape h = shape_of(L.K);
    const int rows = block_rows(h);
    const long long want = ((long long)L.T + rows - 1) / rows;
    // rows of a block's length: what is resident at once; shorter ones: twice that
    // (57600 x 128: their blocks are done sooner than the next row could be asked for)
    int blocks = 8;
    switch (h) {
        case Shape::G128x1: blocks = forward_blocks(128, 1); break;
        case Shape::G256x1: blocks = forward_blocks(256, 1); break;
        case Shape::G256x2: blocks = forward_blocks(256, 2); break;
        case Shape::G512x2: blocks = forward_blocks(512, 2); break;
        case Shape::G512x4: blocks = forward_blocks(512, 4); break;
        case Shape::Long: blocks = 4; break;
        default: break;
    }
    const long long most = (long long)sms * blocks;
    const int grid = (int)(want < most ? want : most);
    const bool q = L.scale != nullptr;
    if (L.type == BVML_F32) {
        return q ? norm_by_shape<float, true>(h, grid, a, s)
                 : norm_by_shape<float, false>(h, grid, a, s);
    } else if (L.type == BVML_F16) {
        return q ? norm_by_shape<__half, true>(h, grid, a, s)
                 : norm_by_shape<__half, false>(h, grid, a, s);
    }
    return q ? norm_by_shape<__nv_bfloat16, true>(h, grid, a, s)
             : norm_by_shape<__nv_bfloat16, false>(h, grid, a, s);
}

// Blocks of the backward pass, each with a row of partial sums: what 148 SMs hold
// at once. A constant and not the device's count, so that the workspace's size
// needs no device.
int norm_backward_parts(int T, int K) {
    const Shape h = shape_of(K);
    int blocks = 1;  // an SM
    switch (h) {
        case Shape::G8:
        case Shape::G16:
        case Shape::G32x1: blocks = backward_blocks(32, 1); break;
        case Shape::G32x2: blocks = backward_blocks(32, 2); break;
        case Shape::G128x1: blocks = backward_blocks(128, 1); break;
        case Shape::G256x1: blocks = backward_blocks(256, 1); break;
        case Shape::G256x2: blocks = backward_blocks(256, 2); break;
        case Shape::G512x2: blocks = backward_blocks(512, 2); break;
        case Shape::G512x4: blocks = backward_blocks(512, 4); break;
        case Shape::Long: blocks = 2; break;
    }
    const long long rows = block_rows(h);
    const long long want = ((long long)T + rows - 1) / rows;
    return (int)(want < 148LL * blocks ? want : 148LL * blocks);
}

cudaError_t launch_rms_norm_backward(const NormBackwardLaunch& L, cudaStream_t s) {
    const int parts = norm_backward_parts(L.T, L.K);
    if (parts > 0) {
        const size_t es = elem_size(L.type);
        NormBwdArgs a{L.dy, L.s, L.w, L.ds, L.dx, L.partial, L.lddy, L.lds, L.ldds, L.lddx,
                      L.T, L.K};
        a.w32 = L.wtype == BVML_F32;
        a.eps = L.eps;
        a.vec = L.K % 8 == 0 && on16(L.dy, L.lddy, es) && on16(L.s, L.lds, es) &&
                (!L.ds || on16(L.ds, L.ldds, es)) && on16(L.w, 0, 1) && on16(L.dx, L.lddx, es);
        const Shape h = shape_of(L.K);
        const cudaError_t e = L.type == BVML_F32 ? norm_backward_by_shape<float>(h, parts, a, s)
                              : L.type == BVML_F16
                                  ? norm_backward_by_shape<__half>(h, parts, a, s)
                                  : norm_backward_by_shape<__nv_bfloat16>(h, parts, a, s);
        if (e != cudaSuccess) return e;
    }
    return launch_column_sum(L.partial, parts, L.K, L.dw, L.wtype, s);
}

cudaError_t launch_column_sum(const float* part, int rows, int cols, void* out, int type,
                              cudaStream_t s) {
    const int grid = (cols + 15) / 16;
    if (type == BVML_F32)
        return launch_pdl(column_sum_kernel<float>, grid, 512, 0, s, true, part, rows, cols,
                          static_cast<float*>(out));
    if (type == BVML_F16)
        return launch_pdl(column_sum_kernel<__half>, grid, 512, 0, s, true, part, rows, cols,
                          static_cast<__half*>(out));
    return launch_pdl(column_sum_kernel<__nv_bfloat16>, grid, 512, 0, s, true, part, rows, cols,
                      static_cast<__nv_bfloat16*>(out));
}

}  // namespace blocks
}  // namespace bvml
