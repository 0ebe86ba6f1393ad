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
//  * warp 0 (in both CTAs) streams operands by TMA in 128-byte swizzled
//    rows of one K step (64 16-bit or 128 8-bit elements) through a ring; the bytes
//    of both CTAs are counted on the first CTA's barrier;
//  * warp 1 of the first CTA issues the MMAs of the pair, and hands ring entries
//    back to both producers by multicast commits;
//  * warps 2-9 drain one of two accumulators in TMEM while the other fills, 16
//    columns of a row a lane at a time, and store 32 rows x 128 bytes by TMA.
//
// Operands come in row-major order for the forward pass; the backward pass reads
// the same tensors with the contracted axis outermost (AT, BT) without a
// transposed copy. A second segment of K steps with tensors of its own adds
// the other half of the gated backward's dx.
//
// Every wait is bounded (TileArgs::wait_limit); one that gives up records an error and stops
// the roles of both CTAs. They meet at a cluster barrier, wait for what is still in flight,
// bounded again, and neither leaves or frees TMEM before that.
//
// Bound by the tensor cores where K is long (87 % busy at 4096 x 4096 x 8192, and then
// by the power limit: 8192 x 4096 x 8192 bf16 takes 334 us alone, 1.65 PFLOP/s, and 435
// in a long row of calls), by writing the output where it is short (57600 x 128 -> 576:
// 21.6 us; filling those 66 MB takes 20.6).
#pragma once

#include "blocks_common.cuh"
#include "gemm_internal.h"
#include "tc_pair.cuh"

namespace bvml {
namespace blocks {

constexpr int kTileEpiWarps = 8;  // two for each quarter of the TMEM lanes
constexpr int kTileThreads = 64 + 32 * kTileEpiWarps;
constexpr int kTileMaxStages = 8;
constexpr uint32_t kTileWaitLimit = 1u << 22;
constexpr int kTileSmem = 227 * 1024;
constexpr int kTileBarBytes = 256;

static __device__ int g_tile_error;

// n / d for n < 2^31 by what Division (gemm_internal.h) holds of d
__device__ __forceinline__ uint32_t divide(uint32_t n, Division d) {
    return (uint32_t)(((uint64_t)n * d.mul) >> 32) >> d.shift;
}

// bytes of one ring entry: 128 rows of A, BN / 2 of B, 128 bytes each
template <int BN> constexpr int tile_stage_bytes() { return (128 + BN / 2) * 128; }
// staging of outputs: 32 rows x 128 bytes a warp, two of them where the ring leaves room
template <int BN> constexpr int tile_buffers() { return BN == 256 ? 1 : 2; }
template <int BN> constexpr int tile_staging_bytes() {
    return kTileEpiWarps * 4096 * tile_buffers<BN>();
}
template <int BN> constexpr int tile_stages() {
    constexpr int n = (kTileSmem - 1024 - kTileBarBytes - tile_staging_bytes<BN>()) /
                      tile_stage_bytes<BN>();
    return n < kTileMaxStages ? n : kTileMaxStages;
}
template <int BN> constexpr int tile_smem_bytes() {
    return 1024 + kTileBarBytes + tile_staging_bytes<BN>() +
           tile_stages<BN>() * tile_stage_bytes<BN>();
}

// A lane finishes kW consecutive columns of one row at a time, as they lie in TMEM. The
// output goes through shared memory: a warp's 32 rows x 128 bytes in the 128-byte
// swizzle, written to global memory by one TMA store, whole lines at a time and
// clipped at the edges (stores from registers, 32 bytes of 32 rows each, cost 57600 x
// 128 -> 576 3 us). What a launch's
// kernel cannot meet is left out at compile time and what is rare stands out of line:
// a short K's epilogue is long beside its MMAs.
constexpr int kW = 16;

template <int OUT> struct OutOf;
template <> struct OutOf<BVML_F32> { using T = float; };
template <> struct OutOf<BVML_F16> { using T = __half; };
template <> struct OutOf<BVML_BF16> { using T = __nv_bfloat16; };

__device__ __forceinline__ void st32(void* p, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]),
                 "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}
// kW columns to rows that start on 16 bytes (wide: on 32).
template <typename T>
__device__ __forceinline__ void put_row(T* p, const float (&v)[kW], bool wide) {
    constexpr int kWords = kW * sizeof(T) / 4;
    uint32_t w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
        else w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    }
    if (__builtin_expect(wide, 1)) {
#pragma unroll
        for (int i = 0; i < kWords; i += 8) st32(reinterpret_cast<uint32_t*>(p) + i, w + i);
    } else {
#pragma unroll
        for (int i = 0; i < kWords; i += 4)
            *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(p) + i) =
                make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    }
}

// ... to row r of a warp's staging buffer: 16-byte unit q of the row at q ^ (r & 7),
// so that eight lanes' writes hit all banks once. c: the chunk's place in the row.
template <typename T>
__device__ __forceinline__ void stage_row(uint8_t* buf, int r, int c, const float (&v)[kW]) {
    constexpr int kUnits = kW * sizeof(T) / 16;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        uint4 w;
        if constexpr (sizeof(T) == 4)
            w = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                           __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
        else
            w = make_uint4(pack2<T>(v[8 * i], v[8 * i + 1]), pack2<T>(v[8 * i + 2], v[8 * i + 3]),
                           pack2<T>(v[8 * i + 4], v[8 * i + 5]),
                           pack2<T>(v[8 * i + 6], v[8 * i + 7]));
        *reinterpret_cast<uint4*>(buf + r * 128 + (((c * kUnits + i) ^ (r & 7)) << 4)) = w;
    }
}

template <int n>
__device__ __forceinline__ void act_row(float (&v)[n], int act) {
    if (act == BVML_ACT_NONE) return;
    // the switch outside the loop: the activation is the same for the whole launch
    switch (act) {
#define BVML_ACT_ROW(code)                                                  \
    case code:                                                              \
        _Pragma("unroll") for (int i = 0; i < n; ++i) v[i] = act_f(v[i], code); \
        break;
        BVML_ACT_ROW(BVML_ACT_RELU)
        BVML_ACT_ROW(BVML_ACT_SIGMOID)
        BVML_ACT_ROW(BVML_ACT_TANH)
        BVML_ACT_ROW(BVML_ACT_SILU)
        BVML_ACT_ROW(BVML_ACT_GELU)
#undef BVML_ACT_ROW
        default: break;
    }
}

// kW values of a vector over columns, on 16 bytes
__device__ __forceinline__ void load_cols(const float* p, float (&c)[kW]) {
#pragma unroll
    for (int i = 0; i < kW / 4; ++i) {
        const float4 f = reinterpret_cast<const float4*>(p)[i];
        c[4 * i] = f.x, c[4 * i + 1] = f.y, c[4 * i + 2] = f.z, c[4 * i + 3] = f.w;
    }
}
__device__ __forceinline__ void scale_cols(float (&v)[kW], float s, const float (&c)[kW]) {
#pragma unroll
    for (int i = 0; i < kW; ++i) v[i] *= s * c[i];
}
// kW elements of a residual's row on 16 bytes, as stored
template <typename T>
struct RawRow {
    uint4 q[kW * sizeof(T) / 16];
};
template <typename T>
__device__ __forceinline__ void ask_row(const T* p, RawRow<T>& r) {
#pragma unroll
    for (int i = 0; i < (int)(kW * sizeof(T) / 16); ++i) r.q[i] = reinterpret_cast<const uint4*>(p)[i];
}
template <typename T>
__device__ __forceinline__ void add_row(float (&v)[kW], const RawRow<T>& r) {
#pragma unroll
    for (int i = 0; i < (int)(kW * sizeof(T) / 4); ++i) {
        const uint32_t w = (&r.q[i / 4].x)[i % 4];
        if constexpr (sizeof(T) == 4) {
            v[i] += __uint_as_float(w);
        } else if constexpr (sizeof(T) == 2) {
            const T lo = reinterpret_cast<const T*>(&w)[0], hi = reinterpret_cast<const T*>(&w)[1];
            v[2 * i] += to_f(lo);
            v[2 * i + 1] += to_f(hi);
        }
    }
}

__device__ __forceinline__ void put_one(void* p, long long i, int type, float v) {
    if (type == BVML_BF16) static_cast<__nv_bfloat16*>(p)[i] = from_f<__nv_bfloat16>(v);
    else if (type == BVML_F16) static_cast<__half*>(p)[i] = from_f<__half>(v);
    else static_cast<float*>(p)[i] = v;
}
__device__ __forceinline__ float get_one(const void* p, long long i, int type) {
    if (type == BVML_BF16) return to_f(static_cast<const __nv_bfloat16*>(p)[i]);
    if (type == BVML_F16) return to_f(static_cast<const __half*>(p)[i]);
    return static_cast<const float*>(p)[i];
}

// One output element of row m, column n from its accumulators (what the backward
// pass keeps of it is stored).
template <bool GATED>
__device__ __forceinline__ float value_one(const TileArgs& a, long long m, int n, float v,
                                           float u) {
    if (a.col_scale[0]) {
        const float rs = a.row_scale[m];
        v *= rs * a.col_scale[0][n];
        if (GATED) u *= rs * a.col_scale[1][n];
    }
    if (GATED) {
        if (a.save[0]) {
            put_one(a.save[0], m * a.lds[0] + n, a.out_type, v);
            put_one(a.save[1], m * a.lds[1] + n, a.out_type, u);
        }
        return act_f(v, a.act) * u;
    }
    if (a.bias) v += a.bias[n];
    if (a.save[0]) put_one(a.save[0], m * a.lds[0] + n, a.out_type, v);
    v = act_f(v, a.act);
    if (a.residual) v += get_one(a.residual, m * a.ldr + n, a.out_type);
    return v;
}

// Chunks at the right edge: one element after the other, out of line.
template <bool GATED>
__device__ __noinline__ void finish_slowly(const TileArgs& a, int m, int n, float* v,
                                           const float* u) {
    const int left = a.N - n < kW ? a.N - n : kW;
    for (int i = 0; i < left; ++i)
        v[i] = value_one<GATED>(a, m, n + i, v[i], GATED ? u[i] : 0.0f);
}

// Epilogue of columns n .. n + kW - 1 of row m, all inside, v <- their
// outputs; raw: the residual's, c: the columns' scales (the gate's) or, without any,
// biases. GRAD: a backward product, whose output is the sum itself.
template <bool F8, bool GATED, bool GRAD, int OUT>
__device__ __forceinline__ void finish_row(const TileArgs& a, int m, int n, float (&v)[kW],
                                           float (&u)[GATED ? kW : 1], float row_scale,
                                           const RawRow<typename OutOf<OUT>::T>& raw,
                                           float (&c)[kW]) {
    using T = typename OutOf<OUT>::T;
    if constexpr (F8) {
        scale_cols(v, row_scale, c);
        if constexpr (GATED) {
            load_cols(a.col_scale[1] + n, c);
            scale_cols(u, row_scale, c);
        } else if (a.bias) {
            load_cols(a.bias + n, c);
        }
    }
    if constexpr (GATED) {
        if (__builtin_expect(a.save[0] != nullptr, 0)) {
            put_row(static_cast<T*>(a.save[0]) + m * a.lds[0] + n, v, a.vec & kWideSave);
            put_row(static_cast<T*>(a.save[1]) + m * a.lds[1] + n, u, a.vec & kWideSave);
        }
        act_row(v, a.act);
#pragma unroll
        for (int i = 0; i < kW; ++i) v[i] *= u[i];
    } else if constexpr (!GRAD) {
        if (a.bias) {
#pragma unroll
            for (int i = 0; i < kW; ++i) v[i] += c[i];
        }
        if (__builtin_expect(a.save[0] != nullptr, 0))
            put_row(static_cast<T*>(a.save[0]) + m * a.lds[0] + n, v, a.vec & kWideSave);
        act_row(v, a.act);
        if (a.residual) add_row(v, raw);
    }
}

// n floats from p + at on 16 bytes; what lies at or past `end` reads zero.
template <int n>
__device__ __forceinline__ void load_some(const float* p, int at, int end, float (&c)[n]) {
    if (__builtin_expect(at + n <= end, 1)) {
#pragma unroll
        for (int i = 0; i < n / 4; ++i) {
            const float4 f = reinterpret_cast<const float4*>(p + at)[i];
            c[4 * i] = f.x, c[4 * i + 1] = f.y, c[4 * i + 2] = f.z, c[4 * i + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < n; ++i) c[i] = at + i < end ? p[at + i] : 0.0f;
    }
}

// A whole box (32 rows x 128 bytes of output) of a product that is not gated, adds no
// residual and keeps nothing, rows on 16 bytes: all its columns at once, without the
// chunks' loop. us, and by chunks: 57600 x 128 -> 576 21.6 (32), with relu 25 (38.5), gelu
// 49 (58). With a residual it is no faster: 55 (57; 49 through shared memory in whole
// lines, which costs the others 4). read(): called when TMEM has been read.
template <bool F8, bool GRAD, int OUT, typename Read>
__device__ __forceinline__ void whole_box(const TileArgs& a, uint32_t acc, int n, float row_scale,
                                          uint8_t* box, int lane, Read read) {
    using T = typename OutOf<OUT>::T;
    constexpr int kBox = 128 / sizeof(T);
    uint32_t x[kBox];
#pragma unroll
    for (int i = 0; i < kBox; i += 32) tc::tmem_ld_32cols(acc + i, x + i);
    float c[kBox] = {};
    if constexpr (F8) load_some(a.col_scale[0], n, a.N, c);
    else if (!GRAD && a.bias) load_some(a.bias, n, a.N, c);
    tc::tmem_ld_wait();
    read();
    float v[kBox];
#pragma unroll
    for (int i = 0; i < kBox; ++i) {
        v[i] = __uint_as_float(x[i]);
        if constexpr (F8) v[i] *= row_scale * c[i];
        else if constexpr (!GRAD) v[i] += c[i];
    }
    if constexpr (F8) {
        if (a.bias) {
            load_some(a.bias, n, a.N, c);
#pragma unroll
            for (int i = 0; i < kBox; ++i) v[i] += c[i];
        }
    }
    if constexpr (!GRAD) act_row(v, a.act);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint4 w;
        if constexpr (sizeof(T) == 4)
            w = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                           __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
        else
            w = make_uint4(pack2<T>(v[8 * i], v[8 * i + 1]), pack2<T>(v[8 * i + 2], v[8 * i + 3]),
                           pack2<T>(v[8 * i + 4], v[8 * i + 5]),
                           pack2<T>(v[8 * i + 6], v[8 * i + 7]));
        *reinterpret_cast<uint4*>(box + lane * 128 + ((i ^ (lane & 7)) << 4)) = w;
    }
}

template <int BN, bool AT, bool BT, bool F8, bool GATED, int OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kTileThreads, 1)
gemm_tile_kernel(const __grid_constant__ TileMaps maps, const TileArgs a) {
    static_assert(!BT || BN % 128 == 0, "a box of B's rows is 64 wide");
    static_assert(BN % 64 == 0, "columns in boxes of 64");
    static_assert(!F8 || (!AT && !BT), "8-bit operands are row-major");
    constexpr int kStage = tile_stage_bytes<BN>();
    constexpr int kStages = tile_stages<BN>();
    constexpr int kStep = F8 ? 128 : 64;  // elements of a K step
    constexpr uint32_t kCols = BN > 128 ? 512 : 2 * BN;  // two accumulators, a power of two
    constexpr int kCN = GATED ? BN / 2 : BN;  // output columns of a tile
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const uint32_t sbase = tc::smem_u32(smem);
    uint8_t* bar_mem = smem + kStages * kStage + tile_staging_bytes<BN>();
    const uint32_t bars = tc::smem_u32(bar_mem);
    const uint32_t bar_full = bars;               // kTileMaxStages, counted on the first CTA's
    const uint32_t bar_empty = bars + 64;         // kTileMaxStages, in each CTA
    const uint32_t bar_acc_full = bars + 128;     // 2, in each CTA
    const uint32_t bar_acc_empty = bars + 144;    // 2, the first CTA's
    const uint32_t bar_end = bars + 160;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_mem + 168);
    // words that both CTAs write or read when they tear down
    int* abort_flag = reinterpret_cast<int*>(bar_mem + 172);
    const uint32_t issued = bars + 176;     // ring entries issued by each CTA, the first CTA's
    const uint32_t committed = bars + 184;  // K steps and tiles whose MMAs were, in each CTA

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
    const int lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int tiles = a.tiles_m * a.tiles_n;
    const int works = tiles * a.splits;
    const int steps = a.steps[0] + a.steps[1];
    // work w -> tile row, tile column, K steps [k0, k1); tiles in groups of
    // 2^group tile rows, so that the pairs at work share operands in L2. The
    // divisions are by numbers known to the host (a 64-bit division here cost
    // each role 900 cycles a tile).
    auto work_of = [&](int w, int& m0, int& n0, int& k0, int& k1, int& split) {
        int t = w;
        split = 0, k0 = 0, k1 = steps;
        if (a.splits > 1) {
            split = tiles > 1 ? (int)divide((uint32_t)w, a.by_tiles) : w;
            t = w - split * tiles;
            k0 = (int)((uint32_t)(steps * split) / (uint32_t)a.splits);
            k1 = (int)((uint32_t)(steps * (split + 1)) / (uint32_t)a.splits);
        }
        const int g = (int)divide((uint32_t)t, a.by_group), r = t - (g << a.group) * a.tiles_n;
        const int gm = a.tiles_m - (g << a.group);  // rows of tiles in the last group
        const bool whole = gm >= 1 << a.group;
        const int rn = whole ? r >> a.group : (int)((uint32_t)r / (uint32_t)gm);
        const int rm = r - (whole ? rn << a.group : rn * gm);
        m0 = ((g << a.group) + rm) * 256 + (int)rank * 128;
        n0 = rn * kCN;
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
    __syncwarp();
    if (warp == 1) {
        tc::tmem_alloc_pair(tc::smem_u32(tmem_slot), kCols);
        tc::tmem_relinquish_pair();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::cluster_sync();  // the peer's barriers exist before anything arrives on them
    begin();
    tc::tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

    auto fail = [&](int code) {
        atomicCAS(&g_tile_error, 0, code);  // the first one
        for (uint32_t r = 0; r < 2; ++r) tc::st_cluster(tc::map_to(bars + 172, r), 1);
    };
    auto aborted = [&]() { return *reinterpret_cast<volatile int*>(abort_flag) != 0; };

    // A wait of a whole warp: every lane polls, and they agree.
    auto wait_all = [&](uint32_t bar, uint32_t parity, int code) {
        const bool done = tc::mbar_wait_pipe(bar, parity, a.wait_limit);
        if (__all_sync(0xffffffffu, done)) return true;
        if (lane == 0) fail(code);
        return false;
    };
    auto gone = [&]() { return __any_sync(0xffffffffu, aborted()) != 0; };

    if (warp == 0) {
        // ---------------------------------------------------------- producer
        const uint32_t on = tc::elect_one();
        const uint32_t first_on = rank == 0 ? on : 0;
        int i = 0;  // ring entries issued
        int slot = 0;
        uint32_t parity = 1;  // of the wait for the slot's hand-back: passes at once at first
        bool ok = true;
        const uint32_t full0 = tc::map_to(bar_full, 0);
        for (int w = pair; ok && w < works; w += pairs) {
            int m0, n0, k0, k1, split;
            work_of(w, m0, n0, k0, k1, split);
            if (gone()) break;
            for (int k = k0; k < k1; ++k, ++i) {
                if (!wait_all(bar_empty + 8 * slot, parity, 1)) {
                    ok = false;
                    break;
                }
                const uint32_t full = full0 + 8 * slot;
                const uint32_t sa = sbase + slot * kStage, sb = sa + 128 * 128;
                const int seg = k >= a.steps[0];
                const int x = (k - (seg ? a.steps[0] : 0)) * kStep;
                if (!tc::copy_ok(sa, AT ? m0 : x, 128 / kStep, false, 0) ||
                    !tc::copy_ok(sb, BT ? n0 : x, 128 / kStep, false, 0)) {
                    ok = false;
                    break;
                }
                tc::mbar_expect_tx_on(first_on, bar_full + 8 * slot, 2 * kStage);
                if constexpr (AT) {
                    tc::tma_load_2d_pair(on, sa, &maps.a[seg], full, m0, x);
                    tc::tma_load_2d_pair(on, sa + 8192, &maps.a[seg], full, m0 + 64, x);
                } else {
                    tc::tma_load_2d_pair(on, sa, &maps.a[seg], full, x, m0);
                }
                if constexpr (GATED) {
                    tc::tma_load_2d_pair(on, sb, &maps.b[rank], full, x, n0);
                } else {
                    const int nb = n0 + (int)rank * (BN / 2);
                    if constexpr (BT) {
#pragma unroll
                        for (int c = 0; c < BN / 128; ++c)
                            tc::tma_load_2d_pair(on, sb + c * 8192, &maps.b[seg], full,
                                                 nb + 64 * c, x);
                    } else {
                        tc::tma_load_2d_pair(on, sb, &maps.b[seg], full, x, nb);
                    }
                }
                if (++slot == kStages) slot = 0, parity ^= 1;
            }
        }
        // nothing may still arrive in shared memory when the pair leaves: the last
        // round's entries have been consumed and handed back (to both CTAs), or, where a
        // wait gave up, the teardown below waits for them
        for (int q = i > kStages ? i - kStages : 0; ok && q < i; ++q) {
            uint32_t n = kTileWaitLimit / 1024;
            bool done = false;
            while (!done && n-- && !gone())
                done = __all_sync(0xffffffffu,
                                  tc::mbar_wait_pipe(bar_empty + 8 * (q % kStages),
                                                     (q / kStages) & 1, 1024));
            if (!done && lane == 0) fail(2);
            ok = done;
        }
        if (lane == 0) tc::st_cluster(tc::map_to(issued + 4 * rank, 0), i);
    } else if (warp == 1) {
        if (rank == 0) {
            // ----------------------------------------------------------- MMA
            const uint32_t on = tc::elect_one();
            int slot = 0, tl = 0;
            uint32_t parity = 0;
            int done_steps = 0, done_tiles = 0;
            bool ok = true;
            const uint64_t da0 = AT ? tc::umma_desc_mn_sw128(sbase, 8192)
                                    : tc::umma_desc_k_sw128(sbase);
            const uint64_t db0 = BT ? tc::umma_desc_mn_sw128(sbase + 128 * 128, 8192)
                                    : tc::umma_desc_k_sw128(sbase + 128 * 128);
            for (int w = pair; ok && w < works; w += pairs, ++tl) {
                int m0, n0, k0, k1, split;
                work_of(w, m0, n0, k0, k1, split);
                const int buf = tl & 1, u = tl >> 1;
                if (gone()) break;
                if (u > 0 && !wait_all(bar_acc_empty + 8 * buf, (u - 1) & 1, 3)) break;
                tc::tc_fence_after();
                const uint32_t acc = tmem + buf * BN;
                for (int k = k0; k < k1; ++k) {
                    if (!wait_all(bar_full + 8 * slot, parity, 4)) {
                        ok = false;
                        break;
                    }
                    tc::tc_fence_after();
                    // addresses in a descriptor count 16-byte units
                    const uint64_t da = da0 + (uint32_t)(slot * (kStage >> 4));
                    const uint64_t db = db0 + (uint32_t)(slot * (kStage >> 4));
#pragma unroll
                    for (int q = 0; q < 4; ++q)  // 32 bytes of K, or 16 rows of k
                        tc::umma_pair<F8>(on, acc, da + q * (AT ? 128 : 2),
                                          db + q * (BT ? 128 : 2), a.idesc, k > k0 || q > 0);
                    tc::umma_commit_pair(on, bar_empty + 8 * slot);
                    ++done_steps;
                    if (++slot == kStages) slot = 0, parity ^= 1;
                }
                if (ok) {
                    tc::umma_commit_pair(on, bar_acc_full + 8 * buf);
                    ++done_tiles;
                }
            }
            // every issued MMA has completed, after an abort too
            tc::umma_commit_pair_local(on, bar_end);
            if (!tc::mbar_wait(bar_end, 0, kTileWaitLimit)) fail(5);
            __syncwarp();
            if (lane < 2) {
                tc::st_cluster(tc::map_to(committed, lane), done_steps);
                tc::st_cluster(tc::map_to(committed + 4, lane), done_tiles);
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue
        const int quarter = warp & 3;            // the TMEM lanes this warp may read
        using T = typename OutOf<OUT>::T;
        static_assert(kTileEpiWarps == 8, "two warps a quarter of the TMEM lanes");
        const int part = (warp - 2) >> 2;        // even or odd boxes of 128-byte rows
        constexpr int kBox = 128 / sizeof(T);    // columns of a box
        constexpr int kBoxes = kCN / kBox;
        static_assert(kCN % kBox == 0, "whole boxes");
        constexpr int kBufs = tile_buffers<BN>();
        uint8_t* stg = smem + kStages * kStage + (warp - 2) * 4096 * kBufs;
        int filled = 0;  // boxes staged by this warp
        const uint32_t acc_empty0 = tc::map_to(bar_acc_empty, 0);
        const bool whole = !GATED && !a.slab && !a.save[0] && !a.residual;
        const bool ahead = !GATED && !BT && a.residual;
        const float* cols = BT || whole ? nullptr : F8 ? a.col_scale[0] : a.bias;
        int tl = 0;
        for (int w = pair; w < works; w += pairs, ++tl) {
            int m0, n0, k0, k1, split;
            work_of(w, m0, n0, k0, k1, split);
            const int mw = m0 + quarter * 32, m = mw + lane;
            const bool in = m < a.M;
            // an odd box falls to either warp in turn
            const int first = kBoxes % 2 ? (part + tl) & 1 : part;
            // The next chunk's residual and scales or biases are on their way while one is
            // finished.
            RawRow<T> raw{};
            float cnext[kW] = {};
            auto ask = [&](int n) {
                if (n + kW > a.N) return;
                if (ahead && in) ask_row(static_cast<const T*>(a.residual) + m * a.ldr + n, raw);
                if (cols) load_cols(cols + n, cnext);
            };
            if (first < kBoxes) ask(n0 + first * kBox);
            const float row_scale = F8 && in ? a.row_scale[m] : 0.0f;
            const int buf = tl & 1, u = tl >> 1;
            if (!wait_all(bar_acc_full + 8 * buf, u & 1, 6) || gone()) break;
            tc::tc_fence_after();
            const uint32_t acc = tmem + buf * BN + ((uint32_t)(quarter * 32) << 16);
            auto hand_back = [&]() {  // this warp is done with the accumulator
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive_cluster_relaxed(acc_empty0 + 8 * buf);
            };
            if (first >= kBoxes) hand_back();
#pragma unroll 1
            for (int b = first; b < kBoxes; b += 2) {
                uint8_t* box = stg + (filled % kBufs) * 4096;
                // the store that last read this buffer has done so
                if (lane == 0) tc::bulk_wait_read<kBufs - 1>();
                __syncwarp();
                const bool done = b + 2 >= kBoxes;
                if (!GATED && whole)
                    whole_box<F8, BT, OUT>(a, acc + b * kBox, n0 + b * kBox, row_scale, box, lane,
                                           [&]() { if (done) hand_back(); });
#pragma unroll 1
                for (int c = 0; c < kBox && !whole; c += kW) {
                    const int n = n0 + b * kBox + c;
                    float v[kW], g[GATED ? kW : 1], cnow[kW];
                    __syncwarp();  // lanes may have gone different ways
                    {
                        uint32_t x[kW], y[GATED ? kW : 1];
                        tc::tmem_ld_16cols(acc + b * kBox + c, x);
                        if constexpr (GATED) tc::tmem_ld_16cols(acc + BN / 2 + b * kBox + c, y);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < kW; ++i) v[i] = __uint_as_float(x[i]);
                        if constexpr (GATED) {
#pragma unroll
                            for (int i = 0; i < kW; ++i) g[i] = __uint_as_float(y[i]);
                        }
                    }
                    const bool last = c + kW == kBox;
                    if (last && done) hand_back();
#pragma unroll
                    for (int i = 0; i < kW; ++i) cnow[i] = cnext[i];
                    const RawRow<T> now = raw;
                    if (!last) ask(n + kW);
                    else if (!done) ask(n0 + (b + 2) * kBox);
                    if (n >= a.N) continue;
                    if (!GATED && a.slab) {  // one of several shares of K, its pitch a multiple of 32
                        if (in)
                            put_row(a.slab + ((long long)split * a.M + m) * a.ldslab + n, v, true);
                        continue;
                    }
                    if (__builtin_expect(n + kW <= a.N, 1)) {
                        if (in)
                            finish_row<F8, GATED, BT, OUT>(a, m, n, v, g, row_scale, now, cnow);
                    } else if (in) {
                        // copies: an array whose address leaves lives in memory everywhere
                        float tv[kW], tg[GATED ? kW : 1];
#pragma unroll
                        for (int i = 0; i < kW; ++i) tv[i] = v[i];
#pragma unroll
                        for (int i = 0; i < (GATED ? kW : 1); ++i) tg[i] = g[i];
                        finish_slowly<GATED>(a, m, n, tv, tg);
#pragma unroll
                        for (int i = 0; i < kW; ++i) v[i] = tv[i];
                    }
                    stage_row<T>(box, lane, c / kW, v);
                }
                if (!GATED && a.slab) continue;
                tc::fence_proxy_async_smem();
                __syncwarp();
                const int n = n0 + b * kBox;
                const bool second = AT && a.out2 && mw >= a.rows1;
                const int row = second ? mw - a.rows1 : mw;
                if (lane == 0) {
                    if (n < a.N && row < a.out_rows &&
                        tc::copy_ok(tc::smem_u32(box), n, sizeof(T), true, row))
                        tc::tma_store_2d(&maps.o[second], tc::smem_u32(box), n, row);
                    tc::bulk_commit();
                }
                ++filled;
            }
        }
        if (lane == 0) tc::bulk_wait_all();  // before shared memory goes
    }
    __syncthreads();
    // The pair's MMAs and stores are done, and, unless a wait gave up, its copies and
    // arrivals.
    tc::cluster_sync();
    if (warp == 0 && gone()) {
        const volatile int* words = reinterpret_cast<volatile int*>(bar_mem + 176);
        // arrivals of the MMAs' commits on this CTA's barriers
        const int steps_done = words[2], tiles_done = words[3];
        for (int q = steps_done > kStages ? steps_done - kStages : 0; q < steps_done; ++q)
            tc::mbar_wait_landed(bar_empty + 8 * (q % kStages), (q / kStages) & 1);
        for (int j = tiles_done > 2 ? tiles_done - 2 : 0; j < tiles_done; ++j)
            tc::mbar_wait_landed(bar_acc_full + 8 * (j & 1), (j >> 1) & 1);
        // Copies of both CTAs, counted here: entries before the last kStages that either
        // issued have been consumed. One that only one CTA issued is made up to what its
        // phase expects.
        const int n0 = words[0], n1 = words[1], n = n0 > n1 ? n0 : n1;
        for (int q = rank == 0 ? (n > kStages ? n - kStages : 0) : n; q < n; ++q) {
            const uint32_t full = bar_full + 8 * (q % kStages);
            if (lane == 0 && q >= n0) tc::mbar_expect_tx(full, kStage);
            if (lane == 0 && q >= n1) tc::mbar_complete_tx(full, kStage);
            __syncwarp();
            tc::mbar_wait_landed(full, (q / kStages) & 1);
        }
    }
    __syncwarp();
    if (warp == 1) tc::tmem_dealloc_pair(tmem, kCols);
    tc::cluster_sync();
}

template <int BN, bool AT, bool BT, bool F8, bool GATED, int OUT>
cudaError_t launch_tile_out(const TileMaps& maps, const TileArgs& a, int pairs, cudaStream_t s) {
    auto kern = gemm_tile_kernel<BN, AT, BT, F8, GATED, OUT>;
    constexpr int smem = tile_smem_bytes<BN>();
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    return launch_pdl(kern, 2 * pairs, kTileThreads, smem, s, true, maps, a);
}
template <int BN, bool AT, bool BT, bool F8, bool GATED>
cudaError_t launch_tile(const TileMaps& maps, const TileArgs& a, int pairs, cudaStream_t s) {
    if (a.out_type == BVML_BF16)
        return launch_tile_out<BN, AT, BT, F8, GATED, BVML_BF16>(maps, a, pairs, s);
    if (a.out_type == BVML_F16)
        return launch_tile_out<BN, AT, BT, F8, GATED, BVML_F16>(maps, a, pairs, s);
    if constexpr (!BT)  // gradients are of the operands' type
        return launch_tile_out<BN, AT, BT, F8, GATED, BVML_F32>(maps, a, pairs, s);
    return cudaErrorInvalidValue;
}

// Host reader of this translation unit's error word; resets it.
// Checked builds: or 1000 and what the checks recorded.
#define BVML_TILE_ERROR_READER(fn)                                             \
    BVML_CHECK_READER(fn##_checks)                                             \
    cudaError_t fn(int* word) {                                                \
        cudaError_t e = cudaMemcpyFromSymbol(word, g_tile_error, sizeof(int)); \
        if (e != cudaSuccess) return e;                                        \
        const int zero = 0;                                                    \
        if (*word) e = cudaMemcpyToSymbol(g_tile_error, &zero, sizeof(int));   \
        if (const unsigned c = fn##_checks(true)) *word = 1000 + (int)c;       \
        return e;                                                              \
    }

}  // namespace blocks
}  // namespace bvml
