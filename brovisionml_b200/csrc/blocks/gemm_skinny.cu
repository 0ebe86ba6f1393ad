// Products with few rows (decoding: one to 128 tokens), bound by reading the
// weights once: out[t, n] = sum_k w[n, k] x[t, k].
//
// The weights are the MMA's 128 rows and the tokens its columns (16 to 128), so
// that one token costs no more tensor-core time than sixteen and every byte that a
// CTA loads is weight. To have enough loads in flight with few weight rows, K is
// shared out over a cluster of up to eight CTAs; each leaves its 128 x tokens fp32
// partial sums in its shared memory, and every CTA adds up a share of the rows over
// the cluster through distributed shared memory, in the order of the ranks
// (no atomics, no workspace, one launch). Gated: a CTA takes 64 rows of each
// projection, and pairs them up where it adds.
//
// us (and TB/s of weights and rows), weights not in L2: 1 x 4096 -> 4096 bf16 10.2
// (3.3), 16 x 4096 -> 12288 20.5 (4.9), 61 x 4096 -> 12288 in 8 bits 16.3 (3.2), gated
// 16 x 4096 -> 11264 33.7 (5.5). What is above the stream is fixed: the launch, the first
// loads' latency, and the sum over the cluster, about 5 us together.
#include "gemm_tile.cuh"

namespace bvml {
namespace blocks {
namespace {

constexpr int kSkinnyThreads = 256;
constexpr int kSkinnyPitch = 132;  // floats between two tokens' partial sums

template <int TOK> constexpr int skinny_stage_bytes() { return (128 + TOK) * 128; }
template <int TOK> constexpr int skinny_stages() {
    // three CTAs an SM with up to 64 tokens, two with more: 72 and 96 KB
    return (TOK <= 64 ? 73728 : 98304) / skinny_stage_bytes<TOK>();
}
template <int TOK> constexpr int skinny_smem_bytes() {
    // 1024-aligned ring (the partial sums take its place), barriers
    return 1024 + skinny_stages<TOK>() * skinny_stage_bytes<TOK>() + 256;
}

// What the epilogue of four neighbouring features of a token reads beside their
// sums; asked for before the cluster meets, so that its latency passes meanwhile.
struct Beside {
    float rs, cs[4], cu[4], add[4], res[4];
};
template <bool GATED>
__device__ __forceinline__ void ask_beside(const TileArgs& a, long long m, int n, Beside& o) {
    if (a.col_scale[0]) o.rs = a.row_scale[m];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (n + e >= a.N) break;
        if (a.col_scale[0]) {
            o.cs[e] = a.col_scale[0][n + e];
            if (GATED) o.cu[e] = a.col_scale[1][n + e];
        }
        if (!GATED && a.bias) o.add[e] = a.bias[n + e];
        if (!GATED && a.residual) o.res[e] = get_one(a.residual, m * a.ldr + n + e, a.out_type);
    }
}
__device__ __forceinline__ void put_four(void* p, long long at, int type, const float (&v)[4],
                                         int left, bool vec) {
    if (vec && left >= 4) {
        if (type == BVML_F32)
            *reinterpret_cast<float4*>(static_cast<float*>(p) + at) =
                make_float4(v[0], v[1], v[2], v[3]);
        else
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + at) =
                type == BVML_BF16 ? make_uint2(pack2<__nv_bfloat16>(v[0], v[1]),
                                               pack2<__nv_bfloat16>(v[2], v[3]))
                                  : make_uint2(pack2<__half>(v[0], v[1]), pack2<__half>(v[2], v[3]));
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (e < left) put_one(p, at + e, type, v[e]);
    }
}

// This CTA's share of the features, summed over the cluster's SPLIT CTAs and
// finished: four neighbouring features of a token a thread, P tokens at a time, all
// the shares' loads in flight at once. The cluster meets between asking for what
// lies beside the first sums and reading them.
template <int SPLIT, bool GATED>
__device__ __forceinline__ void add_up(const TileArgs& a, uint32_t sbase, int rank, int f0, int t0,
                                       int tok) {
    constexpr int kShare = (GATED ? 64 : 128) / SPLIT;
    constexpr int kQuads = kShare / 4;
    constexpr int P = SPLIT * (GATED ? 2 : 1) <= 4 ? 2 : 1;
    const int toks = a.M - t0 < tok ? a.M - t0 : tok;
    const int items = kQuads * toks;
    const bool vec = a.vec & kOn16;
    Beside b[P];
    auto ask = [&](int i0) {
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int i = i0 + p * kSkinnyThreads;
            if (i < items)
                ask_beside<GATED>(a, t0 + i / kQuads, f0 + rank * kShare + i % kQuads * 4, b[p]);
        }
    };
    ask(threadIdx.x);
    tc::cluster_sync();
    uint32_t base[SPLIT];
#pragma unroll
    for (int r = 0; r < SPLIT; ++r) base[r] = tc::map_to(sbase, r);
    for (int i0 = threadIdx.x; i0 < items; i0 += P * kSkinnyThreads) {
        if (i0 != (int)threadIdx.x) ask(i0);
        float4 x[P][SPLIT], y[P][GATED ? SPLIT : 1];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            // past the end: the first item's place again, not used
            const int i = i0 + p * kSkinnyThreads < items ? i0 + p * kSkinnyThreads : i0;
            const uint32_t at =
                4 * (i / kQuads * kSkinnyPitch + rank * kShare + i % kQuads * 4);
#pragma unroll
            for (int r = 0; r < SPLIT; ++r) {
                x[p][r] = tc::ld_cluster4(base[r] + at);
                if constexpr (GATED) y[p][r] = tc::ld_cluster4(base[r] + at + 4 * 64);
            }
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int i = i0 + p * kSkinnyThreads;
            if (i >= items) break;
            float v[4] = {x[p][0].x, x[p][0].y, x[p][0].z, x[p][0].w}, u[4] = {};
#pragma unroll
            for (int r = 1; r < SPLIT; ++r)
                v[0] += x[p][r].x, v[1] += x[p][r].y, v[2] += x[p][r].z, v[3] += x[p][r].w;
            if constexpr (GATED) {
                u[0] = y[p][0].x, u[1] = y[p][0].y, u[2] = y[p][0].z, u[3] = y[p][0].w;
#pragma unroll
                for (int r = 1; r < SPLIT; ++r)
                    u[0] += y[p][r].x, u[1] += y[p][r].y, u[2] += y[p][r].z, u[3] += y[p][r].w;
            }
            const long long m = t0 + i / kQuads;
            const int n = f0 + rank * kShare + i % kQuads * 4, left = a.N - n;
            if (left <= 0) continue;
            if (a.col_scale[0]) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] *= b[p].rs * b[p].cs[e];
                    if (GATED) u[e] *= b[p].rs * b[p].cu[e];
                }
            }
            if (!GATED && a.bias) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += b[p].add[e];
            }
            if (a.save[0]) {
                put_four(a.save[0], m * a.lds[0] + n, a.out_type, v, left, vec);
                if (GATED) put_four(a.save[1], m * a.lds[1] + n, a.out_type, u, left, vec);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = act_f(v[e], a.act);
                if (GATED) v[e] *= u[e];
                if (!GATED && a.residual) v[e] += b[p].res[e];
            }
            put_four(a.out, m * a.ldo + n, a.out_type, v, left, vec);
        }
    }
}

template <int TOK, bool F8, bool GATED>
__global__ void __launch_bounds__(kSkinnyThreads, TOK <= 64 ? 3 : 2)  // what shared memory holds
skinny_kernel(const __grid_constant__ TileMaps maps, const SkinnyArgs sa) {
    constexpr int kStage = skinny_stage_bytes<TOK>();
    constexpr int kStages = skinny_stages<TOK>();
    static_assert(TOK * kSkinnyPitch * 4 <= kStages * kStage, "partial sums fit the ring");
    constexpr int kStep = F8 ? 128 : 64;
    constexpr uint32_t kCols = TOK < 32 ? 32 : TOK;
    constexpr int kFeatures = GATED ? 64 : 128;
    const TileArgs& a = sa.t;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const uint32_t sbase = tc::smem_u32(smem);
    uint8_t* bar_mem = smem + kStages * kStage;
    const uint32_t bar_full = tc::smem_u32(bar_mem), bar_empty = bar_full + 64,
                   bar_acc = bar_full + 128;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_mem + 136);

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    const int split = sa.split;
    const int rank = blockIdx.x % split;  // the cluster's CTAs are neighbours in x
    const int f0 = (blockIdx.x / split) * kFeatures, t0 = blockIdx.y * TOK;
    const int k0 = (int)((long long)a.steps[0] * rank / split);
    const int k1 = (int)((long long)a.steps[0] * (rank + 1) / split);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            tc::mbar_init(bar_full + 8 * s, 1);
            tc::mbar_init(bar_empty + 8 * s, 1);
        }
        tc::mbar_init(bar_acc, 1);
        tc::mbar_fence_init();
    }
    __syncwarp();
    if (warp == 1) {
        tc::tmem_alloc(tc::smem_u32(tmem_slot), kCols);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    // begin(), with the first weights asked for (as many as the ring holds) in between:
    // they come to L2 while the kernel before ends (8-bit, 61 rows: 17.2 -> 16.3 us; all
    // of them at once cost 64 x 8192 -> 8192 30.2 -> 38 us).
    pdl_trigger();
    if (warp == 0) {
        const uint32_t on = tc::elect_one();
        for (int k = k0; k < k1 && k < k0 + kStages; ++k) {
            tc::tma_prefetch_2d(on, &maps.b[0], k * kStep, f0);
            if constexpr (GATED) tc::tma_prefetch_2d(on, &maps.b[1], k * kStep, f0);
        }
    }
    pdl_wait();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

    auto fail = [&](int code) { atomicCAS(&g_tile_error, 0, code); };
    auto wait_all = [&](uint32_t bar, uint32_t parity, uint32_t limit, int code) {  // a warp's
        const bool done = tc::mbar_wait_pipe(bar, parity, limit);
        if (__all_sync(0xffffffffu, done)) return true;
        if (lane == 0) fail(code);
        return false;
    };
    if (warp == 0) {
        const uint32_t on = tc::elect_one();
        int i = 0, slot = 0;
        uint32_t phase = 1;
        for (int k = k0; k < k1; ++k, ++i) {
            if (!wait_all(bar_empty + 8 * slot, phase, a.wait_limit, 11)) break;
            const uint32_t d = sbase + slot * kStage;
            if (!tc::copy_ok(d, k * kStep, 128 / kStep, false, 0)) break;
            tc::mbar_expect_tx_on(on, bar_full + 8 * slot, kStage);
            tc::tma_load_2d(on, d, &maps.b[0], bar_full + 8 * slot, k * kStep, f0);
            if constexpr (GATED)
                tc::tma_load_2d(on, d + 8192, &maps.b[1], bar_full + 8 * slot, k * kStep, f0);
            tc::tma_load_2d(on, d + 128 * 128, &maps.a[0], bar_full + 8 * slot, k * kStep, t0);
            if (++slot == kStages) slot = 0, phase ^= 1;
        }
        // no copy may still be landing when the ring is used anew
        for (int q = i > kStages ? i - kStages : 0; q < i; ++q)
            if (!wait_all(bar_full + 8 * (q % kStages), (q / kStages) & 1, kTileWaitLimit, 12)) break;
    } else if (warp == 1) {
        const uint32_t on = tc::elect_one();
        int slot = 0;
        uint32_t phase = 0;
        const uint64_t dw0 = tc::umma_desc_k_sw128(sbase);
        const uint64_t dx0 = tc::umma_desc_k_sw128(sbase + 128 * 128);
        for (int k = k0; k < k1; ++k) {
            if (!wait_all(bar_full + 8 * slot, phase, a.wait_limit, 13)) break;
            tc::tc_fence_after();
            const uint64_t dw = dw0 + (uint32_t)(slot * (kStage >> 4));
            const uint64_t dx = dx0 + (uint32_t)(slot * (kStage >> 4));
#pragma unroll
            for (int q = 0; q < 4; ++q)
                tc::umma_single<F8>(on, tmem, dw + 2 * q, dx + 2 * q, a.idesc, k > k0 || q > 0);
            tc::umma_commit_on(on, bar_empty + 8 * slot);
            if (++slot == kStages) slot = 0, phase ^= 1;
        }
        tc::umma_commit_on(on, bar_acc);
    }
    __syncwarp();
    // the accumulator, and with it every copy and MMA, is complete
    if (!tc::mbar_wait(bar_acc, 0, kTileWaitLimit)) fail(14);
    __syncthreads();  // ... also the producer's look at its last copies
    __syncwarp();
    tc::tc_fence_after();
    // partial[token][row]: a lane is a row, so a warp writes 32 neighbours
    float* partial = reinterpret_cast<float*>(smem);
    {
        const int quarter = warp & 3, half = warp >> 2;
        constexpr int kPer = TOK < 32 ? 16 : TOK / 2;  // columns of a warp
        if (half * kPer < TOK) {
#pragma unroll
            for (int c = 0; c < kPer; c += 16) {
                uint32_t v[16];
                tc::tmem_ld_16cols(tmem + ((uint32_t)(quarter * 32) << 16) + half * kPer + c, v);
                tc::tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    partial[(half * kPer + c + e) * kSkinnyPitch + quarter * 32 + lane] =
                        __uint_as_float(v[e]);
            }
        }
        tc::tc_fence_before();
    }
    __syncthreads();
    __syncwarp();
    if (warp == 1) tc::tmem_dealloc(tmem, kCols);
    __syncwarp();
    switch (split) {
        case 1: add_up<1, GATED>(a, sbase, rank, f0, t0, TOK); break;
        case 2: add_up<2, GATED>(a, sbase, rank, f0, t0, TOK); break;
        case 4: add_up<4, GATED>(a, sbase, rank, f0, t0, TOK); break;
        default: add_up<8, GATED>(a, sbase, rank, f0, t0, TOK); break;
    }
    tc::cluster_sync();  // no CTA leaves while another still reads its sums
}

template <int TOK, bool F8, bool GATED>
cudaError_t launch_one(const TileMaps& m, const SkinnyArgs& a, cudaStream_t s) {
    auto kern = skinny_kernel<TOK, F8, GATED>;
    constexpr int smem = skinny_smem_bytes<TOK>();
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    constexpr int kFeatures = GATED ? 64 : 128;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((a.t.N + kFeatures - 1) / kFeatures * a.split),
                       (unsigned)((a.t.M + TOK - 1) / TOK));
    cfg.blockDim = dim3(kSkinnyThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)a.split;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, m, a);
}

template <bool F8, bool GATED>
cudaError_t by_tokens(int tok, const TileMaps& m, const SkinnyArgs& a, cudaStream_t s) {
    switch (tok) {
        case 16: return launch_one<16, F8, GATED>(m, a, s);
        case 32: return launch_one<32, F8, GATED>(m, a, s);
        case 64: return launch_one<64, F8, GATED>(m, a, s);
        default: return launch_one<128, F8, GATED>(m, a, s);
    }
}

}  // namespace

cudaError_t launch_skinny(int tok, bool f8, bool gated, const TileMaps& m, const SkinnyArgs& a,
                          cudaStream_t s) {
    if (f8) return gated ? by_tokens<true, true>(tok, m, a, s) : by_tokens<true, false>(tok, m, a, s);
    return gated ? by_tokens<false, true>(tok, m, a, s) : by_tokens<false, false>(tok, m, a, s);
}

BVML_TILE_ERROR_READER(skinny_error)

}  // namespace blocks
}  // namespace bvml
