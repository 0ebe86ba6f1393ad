// Matrix products of the feed-forward operators, the simplest form: a 64 x 64
// tile a block, 4 x 4 outputs a thread, fp32 FMAs over 16-wide slices of K in
// shared memory. Takes every layout and stride.
#include "blocks_common.cuh"
#include "blocks_internal.h"

namespace bvml {
namespace blocks {
namespace {

__device__ __forceinline__ float fetch(const void* p, long long i, int type) {
    switch (type) {
        case BVML_F16: return to_f(static_cast<const __half*>(p)[i]);
        case BVML_BF16: return to_f(static_cast<const __nv_bfloat16*>(p)[i]);
        case BVML_E4M3:
            return float(*(reinterpret_cast<const __nv_fp8_e4m3*>(p) + i));
        default: return static_cast<const float*>(p)[i];
    }
}
__device__ __forceinline__ void put(void* p, long long i, int type, float v) {
    switch (type) {
        case BVML_F16: static_cast<__half*>(p)[i] = from_f<__half>(v); break;
        case BVML_BF16: static_cast<__nv_bfloat16*>(p)[i] = from_f<__nv_bfloat16>(v); break;
        default: static_cast<float*>(p)[i] = v;
    }
}

__global__ void __launch_bounds__(256) gemm_kernel(const GemmLaunch L) {
    __shared__ float sa[16][65], sb[2][16][65];
    const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[2][4][4] = {};
    for (int seg = 0; seg < 2; ++seg) {
        const int nb = L.gated ? 2 : 1;
        for (int k0 = 0; k0 < L.k[seg]; k0 += 16) {
            for (int i = threadIdx.x; i < 64 * 16; i += 256) {
                const int r = L.a_t ? i % 64 : i / 16, c = L.a_t ? i / 64 : i % 16;
                const int m = m0 + r, k = k0 + c;
                const long long at = L.a_t ? (long long)k * L.lda[seg] + m
                                           : (long long)m * L.lda[seg] + k;
                sa[c][r] = m < L.M && k < L.k[seg] ? fetch(L.a[seg], at, L.in_type) : 0.0f;
            }
            for (int q = 0; q < nb; ++q) {
                const int src = L.gated ? q : seg;
                for (int i = threadIdx.x; i < 64 * 16; i += 256) {
                    const int r = L.b_t ? i % 64 : i / 16, c = L.b_t ? i / 64 : i % 16;
                    const int n = n0 + r, k = k0 + c;
                    const long long at = L.b_t ? (long long)k * L.ldb[src] + n
                                               : (long long)n * L.ldb[src] + k;
                    sb[q][c][r] = n < L.N && k < L.k[seg] ? fetch(L.b[src], at, L.in_type) : 0.0f;
                }
            }
            __syncthreads();
            for (int q = 0; q < nb; ++q)
                for (int c = 0; c < 16; ++c)
                    for (int i = 0; i < 4; ++i)
                        for (int j = 0; j < 4; ++j)
                            acc[q][i][j] = fmaf(sa[c][ty * 4 + i], sb[q][c][tx * 4 + j],
                                                acc[q][i][j]);
            __syncthreads();
        }
    }
    for (int i = 0; i < 4; ++i) {
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (m >= L.M || n >= L.N) continue;
            const float rs = L.row_scale ? L.row_scale[m] : 1.0f;
            float v = acc[0][i][j] * rs * (L.col_scale[0] ? L.col_scale[0][n] : 1.0f);
            if (L.gated) {
                const float u = acc[1][i][j] * rs * (L.col_scale[1] ? L.col_scale[1][n] : 1.0f);
                if (L.save[0]) {
                    put(L.save[0], m * L.lds[0] + n, L.out_type, v);
                    put(L.save[1], m * L.lds[1] + n, L.out_type, u);
                }
                v = act_f(v, L.act) * u;
            } else {
                if (L.bias) v += L.bias[n];
                if (L.save[0]) put(L.save[0], m * L.lds[0] + n, L.out_type, v);
                v = act_f(v, L.act);
                if (L.residual) v += fetch(L.residual, m * L.ldr + n, L.out_type);
            }
            if (!L.out2 || m < L.rows0) put(L.out, m * L.ldo + n, L.out_type, v);
            else if (m >= L.rows1) put(L.out2, (m - L.rows1) * L.ldo2 + n, L.out_type, v);
        }
    }
}

}  // namespace

size_t gemm_workspace_bytes(const GemmLaunch&) { return 0; }

cudaError_t launch_gemm(const GemmLaunch& L, void*, cudaStream_t s) {
    if (L.M == 0 || L.N == 0) return cudaSuccess;
    const dim3 grid((L.N + 63) / 64, (L.M + 63) / 64);
    if (grid.y > 65535) return cudaErrorInvalidValue;
    gemm_kernel<<<grid, 256, 0, s>>>(L);
    return cudaGetLastError();
}

cudaError_t gemm_errors(int* word) {
    *word = 0;
    return cudaSuccess;
}

}  // namespace blocks
}  // namespace bvml
