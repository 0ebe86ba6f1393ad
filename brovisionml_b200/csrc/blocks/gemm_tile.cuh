// The large matrix products of the feed-forward operators on CTA pairs
// (tcgen05.mma cta_group::2, sm_100a).
//
//   D[m, n] = sum_k A[m, k] B[n, k], fp32 accumulation, then the epilogue
//   act(D row_scale col_scale + bias) + residual, or act(G) U for the gated pair
//
// A pair of CTAs computes 256 rows x BN columns: each CTA stages its own 128 rows
// of A and half of B's rows, and the pair's tensor cores read both halves of B, so
// a CTA loads 128 + BN / 2 rows a K step instead of 128 + BN. Gated: the first
// CTA's half of B is the gate's rows, the second's the up projection's, and one
// accumulator holds both projections of BN / 2 features side by side.
//
// Persistent, one pair on two SMs:
//  * warp 0 (one lane, in both CTAs) streams operands by TMA in 128-byte swizzled
//    rows of one K step (64 16-bit or 128 8-bit elements) through a ring; the bytes
//    of both CTAs are counted on the first CTA's barrier;
//  * warp 1 of the first CTA issues the MMAs of the pair, and hands ring entries
//    back to both producers by multicast commits;
//  * warps 2-9 drain one of two accumulators in TMEM while the other fills: 32
//    columns at a time through a swizzled staging buffer in shared memory, so that a
//    thread finishes eight consecutive columns of a row and loads and stores
//    16 bytes (the residual, the outputs) where the rows allow it.
//
// Operands come in row-major order for the forward pass; the backward pass reads
// the same tensors with the contracted axis outermost (AT, BT) without a
// transposed copy. A second segment of K steps with tensors of its own adds
// the other half of the gated backward's dx.
//
// Every wait is bounded; one that gives up records an error and both CTAs tear
// down, meeting at a cluster barrier before either leaves.
#pragma once

#include "blocks_common.cuh"
#include "gemm_internal.h"
#include "tc_pair.cuh"

namespace bvml {
namespace blocks {

constexpr int kTileThreads = 320;
constexpr int kTileEpiWarps = 8;
constexpr int kTileMaxStages = 8;
constexpr uint32_t kTileWaitLimit = 1u << 22;
constexpr int kTileSmem = 227 * 1024;
constexpr int kTileBarBytes = 256;

static __device__ int g_tile_error;

// bytes of one ring entry: 128 rows of A, BN / 2 of B, 128 bytes each
template <int BN> constexpr int tile_stage_bytes() { return (128 + BN / 2) * 128; }
// staging: 32 rows x 32 fp32 columns a warp, one for each projection
template <bool GATED> constexpr int tile_staging_bytes() {
    return kTileEpiWarps * 4096 * (GATED ? 2 : 1);
}
template <int BN, bool GATED> constexpr int tile_stages() {
    constexpr int n = (kTileSmem - 1024 - kTileBarBytes - tile_staging_bytes<GATED>()) /
                      tile_stage_bytes<BN>();
    return n < kTileMaxStages ? n : kTileMaxStages;
}
template <int BN, bool GATED> constexpr int tile_smem_bytes() {
    return 1024 + kTileBarBytes + tile_staging_bytes<GATED>() +
           tile_stages<BN, GATED>() * tile_stage_bytes<BN>();
}

// The rows of a group that a lane finishes at once: R rows m0, m0 + step, ...
// of eight consecutive columns n .., `left` of them inside the matrix.
template <int R>
struct Group {
    int m0, step, n, left;
};

// Rows past the last are skipped.
template <typename T, int R>
__device__ __forceinline__ void put_rows(T* base, long long ld, const Group<R>& g, int M,
                                         const float (&v)[R][8], bool vec) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int m = g.m0 + i * g.step;
        if (m >= M) continue;
        T* p = base + m * ld + g.n;
        if (vec && g.left >= 8) {
            store8(p, v[i]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < g.left) p[e] = from_f<T>(v[i][e]);
        }
    }
}
template <int R>
__device__ __forceinline__ void put_rows(void* base, long long ld, int type, const Group<R>& g,
                                         int M, const float (&v)[R][8], bool vec) {
    if (type == BVML_BF16) put_rows(static_cast<__nv_bfloat16*>(base), ld, g, M, v, vec);
    else if (type == BVML_F16) put_rows(static_cast<__half*>(base), ld, g, M, v, vec);
    else put_rows(static_cast<float*>(base), ld, g, M, v, vec);
}
template <typename T, int R>
__device__ __forceinline__ void add_rows(const T* base, long long ld, const Group<R>& g, int M,
                                         float (&v)[R][8], bool vec) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int m = g.m0 + i * g.step;
        if (m >= M) continue;
        const T* p = base + m * ld + g.n;
        if (vec && g.left >= 8) {
            float r[8];
            load8(p, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] += r[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < g.left) v[i][e] += to_f(p[e]);
        }
    }
}

template <int R>
__device__ __forceinline__ void act_rows(float (&v)[R][8], int act) {
    // the switch outside the loops: the activation is the same for the whole launch
    switch (act) {
#define BVML_ACT_ROWS(code)                                                          \
    case code:                                                                       \
        _Pragma("unroll") for (int i = 0; i < R; ++i)                                \
            _Pragma("unroll") for (int e = 0; e < 8; ++e) v[i][e] = act_f(v[i][e], code); \
        break;
        BVML_ACT_ROWS(BVML_ACT_RELU)
        BVML_ACT_ROWS(BVML_ACT_SIGMOID)
        BVML_ACT_ROWS(BVML_ACT_TANH)
        BVML_ACT_ROWS(BVML_ACT_SILU)
        BVML_ACT_ROWS(BVML_ACT_GELU)
#undef BVML_ACT_ROWS
        default: break;
    }
}

// Epilogue of a lane's group. Every choice that is the same for the launch is
// made once for all R rows, so that their loads and stores are in flight together.
template <int R, bool GATED>
__device__ __forceinline__ void finish_rows(const TileArgs& a, const Group<R>& g, float (&v)[R][8],
                                            float (&u)[GATED ? R : 1][8]) {
    float c[8];
    if (a.col_scale[0]) {
        float rs[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int m = g.m0 + i * g.step;
            rs[i] = m < a.M ? __ldg(a.row_scale + m) : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = e < g.left ? __ldg(a.col_scale[0] + g.n + e) : 0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] *= rs[i] * c[e];
        if constexpr (GATED) {
#pragma unroll
            for (int e = 0; e < 8; ++e) c[e] = e < g.left ? __ldg(a.col_scale[1] + g.n + e) : 0.0f;
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) u[i][e] *= rs[i] * c[e];
        }
    }
    if constexpr (GATED) {
        if (a.save[0]) {
            put_rows(a.save[0], a.lds[0], a.out_type, g, a.M, v, a.vec & kVecSave);
            put_rows(a.save[1], a.lds[1], a.out_type, g, a.M, u, a.vec & kVecSave);
        }
        act_rows(v, a.act);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] *= u[i][e];
    } else {
        if (a.bias) {
#pragma unroll
            for (int e = 0; e < 8; ++e) c[e] = e < g.left ? __ldg(a.bias + g.n + e) : 0.0f;
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] += c[e];
        }
        if (a.save[0]) put_rows(a.save[0], a.lds[0], a.out_type, g, a.M, v, a.vec & kVecSave);
        act_rows(v, a.act);
        if (a.residual) {
            const bool vec = a.vec & kVecRes;
            if (a.out_type == BVML_BF16)
                add_rows(static_cast<const __nv_bfloat16*>(a.residual), a.ldr, g, a.M, v, vec);
            else if (a.out_type == BVML_F16)
                add_rows(static_cast<const __half*>(a.residual), a.ldr, g, a.M, v, vec);
            else
                add_rows(static_cast<const float*>(a.residual), a.ldr, g, a.M, v, vec);
        }
    }
    if (!a.out2 || g.m0 + (R - 1) * g.step < a.rows0) {
        put_rows(a.out, a.ldo, a.out_type, g, a.M, v, a.vec & kVecOut);
    } else if (g.m0 >= a.rows1) {
        Group<R> h = g;
        h.m0 -= a.rows1;
        put_rows(a.out2, a.ldo2, a.out_type, h, a.M - a.rows1, v, a.vec & kVecOut2);
    } else {  // the few groups that span the border, row by row
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int m = g.m0 + i * g.step;
            Group<1> h{m, 0, g.n, g.left};
            float one[1][8];
#pragma unroll
            for (int e = 0; e < 8; ++e) one[0][e] = v[i][e];
            if (m < a.rows0) {
                put_rows(a.out, a.ldo, a.out_type, h, a.M, one, a.vec & kVecOut);
            } else if (m >= a.rows1) {
                h.m0 -= a.rows1;
                put_rows(a.out2, a.ldo2, a.out_type, h, a.M - a.rows1, one, a.vec & kVecOut2);
            }
        }
    }
}

template <int BN, bool AT, bool BT, bool F8, bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTileThreads, 1)
gemm_tile_kernel(const __grid_constant__ TileMaps maps, const TileArgs a) {
    static_assert(!BT || BN >= 128, "a box of B's rows is 64 wide");
    static_assert(!F8 || (!AT && !BT), "8-bit operands are row-major");
    constexpr int kStage = tile_stage_bytes<BN>();
    constexpr int kStages = tile_stages<BN, GATED>();
    constexpr int kStaging = tile_staging_bytes<GATED>();
    constexpr int kStep = F8 ? 128 : 64;  // elements of a K step
    constexpr uint32_t kCols = 2 * BN;    // two accumulators
    constexpr int kCN = GATED ? BN / 2 : BN;  // output columns of a tile
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const uint32_t sbase = tc::smem_u32(smem);
    uint8_t* bar_mem = smem + kStages * kStage + kStaging;
    const uint32_t bars = tc::smem_u32(bar_mem);
    const uint32_t bar_full = bars;               // kTileMaxStages, counted on the first CTA's
    const uint32_t bar_empty = bars + 64;         // kTileMaxStages, in each CTA
    const uint32_t bar_acc_full = bars + 128;     // 2, in each CTA
    const uint32_t bar_acc_empty = bars + 144;    // 2, the first CTA's
    const uint32_t bar_end = bars + 160;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_mem + 168);
    int* abort_flag = reinterpret_cast<int*>(bar_mem + 172);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int tiles = a.tiles_m * a.tiles_n;
    const int works = tiles * a.splits;
    const int steps = a.steps[0] + a.steps[1];
    // work w -> tile row, tile column, K steps [k0, k1); tiles in groups of
    // kGroup tile rows, so that the pairs at work share operands in L2
    auto work_of = [&](int w, int& m0, int& n0, int& k0, int& k1, int& split) {
        split = w / tiles;
        const int t = w - split * tiles;
        constexpr int kGroup = 8;
        const int per = kGroup * a.tiles_n;
        const int g = t / per, r = t - g * per;
        const int gm = a.tiles_m - g * kGroup < kGroup ? a.tiles_m - g * kGroup : kGroup;
        m0 = (g * kGroup + r % gm) * 256 + (int)rank * 128;
        n0 = (r / gm) * kCN;
        k0 = (int)((long long)steps * split / a.splits);
        k1 = (int)((long long)steps * (split + 1) / a.splits);
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < kTileMaxStages; ++s) {
            tc::mbar_init(bar_full + 8 * s, 1);
            tc::mbar_init(bar_empty + 8 * s, 1);
        }
        for (int q = 0; q < 2; ++q) {
            tc::mbar_init(bar_acc_full + 8 * q, 1);
            tc::mbar_init(bar_acc_empty + 8 * q, 2 * kTileEpiWarps);
        }
        tc::mbar_init(bar_end, 1);
        *abort_flag = 0;
        tc::mbar_fence_init();
        tc::tma_prefetch_desc(&maps.a[0]);
        tc::tma_prefetch_desc(&maps.b[0]);
    }
    if (warp == 1) {
        tc::tmem_alloc_pair(tc::smem_u32(tmem_slot), kCols);
        tc::tmem_relinquish_pair();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync();  // the peer's barriers exist before anything arrives on them
    tc::tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    auto fail = [&](int code) {
        atomicExch(&g_tile_error, code);
        *reinterpret_cast<volatile int*>(abort_flag) = 1;
    };
    auto aborted = [&]() { return *reinterpret_cast<volatile int*>(abort_flag) != 0; };

    if (warp == 0) {
        if (lane == 0) {
            // ------------------------------------------------------ producer
            int i = 0;  // ring entries issued
            bool ok = true;
            for (int w = pair; ok && w < works; w += pairs) {
                int m0, n0, k0, k1, split;
                work_of(w, m0, n0, k0, k1, split);
                for (int k = k0; k < k1; ++k, ++i) {
                    const int s = i % kStages, j = i / kStages;
                    if (j > 0 && !tc::mbar_wait_pipe(bar_empty + 8 * s, (j - 1) & 1,
                                                     kTileWaitLimit)) {
                        fail(1);
                        ok = false;
                        break;
                    }
                    if (aborted()) {
                        ok = false;
                        break;
                    }
                    if (rank == 0) tc::mbar_expect_tx(bar_full + 8 * s, 2 * kStage);
                    const uint32_t full = tc::map_to(bar_full + 8 * s, 0);
                    const uint32_t sa = sbase + s * kStage, sb = sa + 128 * 128;
                    const int seg = k >= a.steps[0];
                    const int x = (k - (seg ? a.steps[0] : 0)) * kStep;
                    if constexpr (AT) {
                        tc::tma_load_2d_pair(sa, &maps.a[seg], full, m0, x);
                        tc::tma_load_2d_pair(sa + 8192, &maps.a[seg], full, m0 + 64, x);
                    } else {
                        tc::tma_load_2d_pair(sa, &maps.a[seg], full, x, m0);
                    }
                    if constexpr (GATED) {
                        tc::tma_load_2d_pair(sb, &maps.b[rank], full, x, n0);
                    } else {
                        const int nb = n0 + (int)rank * (BN / 2);
                        if constexpr (BT) {
#pragma unroll
                            for (int c = 0; c < BN / 128; ++c)
                                tc::tma_load_2d_pair(sb + c * 8192, &maps.b[seg], full,
                                                     nb + 64 * c, x);
                        } else {
                            tc::tma_load_2d_pair(sb, &maps.b[seg], full, x, nb);
                        }
                    }
                }
            }
            // nothing may still arrive in shared memory when the pair leaves: the last
            // round's entries have been consumed and handed back (to both CTAs);
            // after an abort the copies at least have landed (the first CTA's
            // barriers count both CTAs' bytes)
            const int q0 = i > kStages ? i - kStages : 0;
            for (int q = q0; ok && q < i; ++q) {
                if (!tc::mbar_wait(bar_empty + 8 * (q % kStages), (q / kStages) & 1,
                                   kTileWaitLimit)) {
                    fail(2);
                    ok = false;
                }
            }
            if (!ok && rank == 0)
                for (int q = q0; q < i; ++q)
                    if (!tc::mbar_wait(bar_full + 8 * (q % kStages), (q / kStages) & 1,
                                       kTileWaitLimit))
                        break;
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            // ----------------------------------------------------------- MMA
            int i = 0, tl = 0;
            bool ok = true;
            for (int w = pair; ok && w < works; w += pairs, ++tl) {
                int m0, n0, k0, k1, split;
                work_of(w, m0, n0, k0, k1, split);
                const int buf = tl & 1, u = tl >> 1;
                if (u > 0 && !tc::mbar_wait_pipe(bar_acc_empty + 8 * buf, (u - 1) & 1,
                                                 kTileWaitLimit)) {
                    fail(3);
                    break;
                }
                tc::tc_fence_after();
                const uint32_t acc = tmem + buf * BN;
                for (int k = k0; k < k1; ++k, ++i) {
                    const int s = i % kStages;
                    if (!tc::mbar_wait_pipe(bar_full + 8 * s, (i / kStages) & 1, kTileWaitLimit) ||
                        aborted()) {
                        fail(4);
                        ok = false;
                        break;
                    }
                    tc::tc_fence_after();
                    const uint32_t sa = sbase + s * kStage, sb = sa + 128 * 128;
                    const uint64_t da = AT ? tc::umma_desc_mn_sw128(sa, 8192)
                                           : tc::umma_desc_k_sw128(sa);
                    const uint64_t db = BT ? tc::umma_desc_mn_sw128(sb, 8192)
                                           : tc::umma_desc_k_sw128(sb);
#pragma unroll
                    for (int q = 0; q < 4; ++q)  // 32 bytes of K, or 16 rows of k
                        tc::umma_pair<F8>(acc, da + q * (AT ? 128 : 2), db + q * (BT ? 128 : 2),
                                          a.idesc, k > k0 || q > 0);
                    tc::umma_commit_pair(bar_empty + 8 * s);
                }
                if (ok) tc::umma_commit_pair(bar_acc_full + 8 * buf);
            }
            // every issued MMA has completed, after an abort too
            tc::umma_commit_pair_local(bar_end);
            if (!tc::mbar_wait(bar_end, 0, kTileWaitLimit)) fail(5);
        }
    } else {
        // ------------------------------------------------------------ epilogue
        const int quarter = warp & 3;            // the TMEM lanes this warp may read
        const int part = (warp - 2) >> 2;        // which half of the columns
        float* stg = reinterpret_cast<float*>(smem + kStages * kStage +
                                              (warp - 2) * 4096 * (GATED ? 2 : 1));
        const uint32_t acc_empty0 = tc::map_to(bar_acc_empty, 0);
        int tl = 0;
        for (int w = pair; w < works; w += pairs, ++tl) {
            int m0, n0, k0, k1, split;
            work_of(w, m0, n0, k0, k1, split);
            const int buf = tl & 1, u = tl >> 1;
            const bool full = tc::mbar_wait_pipe(bar_acc_full + 8 * buf, u & 1, kTileWaitLimit);
            if (!__all_sync(0xffffffffu, full && !aborted())) {  // the whole warp gives up
                if (lane == 0) fail(6);
                break;
            }
            tc::tc_fence_after();
            const uint32_t acc = tmem + buf * BN + ((uint32_t)(quarter * 32) << 16);
            constexpr int kHalf = kCN / 2;               // columns of this warp
            constexpr int kW = kHalf < 32 ? kHalf : 32;  // ... at a time
#pragma unroll 1
            for (int c = 0; c < kHalf; c += kW) {
                const int col = part * kHalf + c;
                // phase 1: a lane holds kW columns of one row; staged as 16-byte units,
                // unit q of row r at q ^ (r & 7): no bank is hit twice
#pragma unroll
                for (int p = 0; p < (GATED ? 2 : 1); ++p) {
                    float* d = stg + p * 1024;
                    if constexpr (kW == 32) {
                        uint32_t v[32];
                        tc::tmem_ld_32cols(acc + col + p * (BN / 2), v);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int q = 0; q < 8; ++q)
                            *reinterpret_cast<uint4*>(d + lane * 32 + ((q ^ (lane & 7)) << 2)) =
                                make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                    } else {
                        static_assert(kW == 32 || kW == 16, "columns a warp takes at a time");
                        uint32_t v[16];
                        tc::tmem_ld_16cols(acc + col + p * (BN / 2), v);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            *reinterpret_cast<uint4*>(d + lane * 32 + ((q ^ (lane & 7)) << 2)) =
                                make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                    }
                }
                if (c + kW == kHalf) {  // this warp is done with the accumulator
                    tc::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive_cluster(acc_empty0 + 8 * buf);
                }
                __syncwarp();
                // phase 2: a lane finishes eight consecutive columns of R rows
                constexpr int kGroups = kW / 8;  // lanes of a row, and R
                constexpr int kRows = 32 / kGroups;
                const int q = lane % kGroups, r0 = lane / kGroups;
                const Group<kGroups> grp{m0 + quarter * 32 + r0, kRows, n0 + col + q * 8,
                                         a.N - (n0 + col + q * 8)};
                float v[kGroups][8], g[GATED ? kGroups : 1][8];
#pragma unroll
                for (int i = 0; i < kGroups; ++i) {
                    const int r = i * kRows + r0;
#pragma unroll
                    for (int p = 0; p < (GATED ? 2 : 1); ++p) {
                        const float* d = stg + p * 1024 + r * 32;
                        const float4 x = *reinterpret_cast<const float4*>(
                            d + (((2 * q) ^ (r & 7)) << 2));
                        const float4 y = *reinterpret_cast<const float4*>(
                            d + (((2 * q + 1) ^ (r & 7)) << 2));
                        float* o = p == 0 ? v[i] : g[GATED ? i : 0];
                        o[0] = x.x, o[1] = x.y, o[2] = x.z, o[3] = x.w;
                        o[4] = y.x, o[5] = y.y, o[6] = y.z, o[7] = y.w;
                    }
                }
                if (grp.left > 0) {
                    if (a.slab)  // one of several shares of K: joined by a second kernel
                        put_rows(a.slab + (long long)split * a.M * a.ldslab, a.ldslab, grp, a.M,
                                 v, true);
                    else
                        finish_rows<kGroups, GATED>(a, grp, v, g);
                }
                __syncwarp();
            }
        }
    }
    __syncthreads();
    __syncwarp();
    tc::cluster_sync();  // the pair's copies, MMAs and arrivals are all done
    if (warp == 1) tc::tmem_dealloc_pair(tmem, kCols);
    tc::cluster_sync();
}

template <int BN, bool AT, bool BT, bool F8, bool GATED>
cudaError_t launch_tile(const TileMaps& maps, const TileArgs& a, int pairs, cudaStream_t s) {
    auto kern = gemm_tile_kernel<BN, AT, BT, F8, GATED>;
    constexpr int smem = tile_smem_bytes<BN, GATED>();
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    kern<<<2 * pairs, kTileThreads, smem, s>>>(maps, a);
    return cudaGetLastError();
}

// Host reader of this translation unit's error word; resets it.
#define BVML_TILE_ERROR_READER(fn)                                            \
    cudaError_t fn(int* word) {                                               \
        cudaError_t e = cudaMemcpyFromSymbol(word, g_tile_error, sizeof(int)); \
        if (e != cudaSuccess || *word == 0) return e;                         \
        const int zero = 0;                                                   \
        return cudaMemcpyToSymbol(g_tile_error, &zero, sizeof(int));          \
    }

}  // namespace blocks
}  // namespace bvml
