// Planning of the feed-forward operators' matrix products: which kernel, tile and
// share of K, the tensor maps, the operands that have to be laid out anew, and the
// sum over shares of K.
#include <cudaTypedefs.h>

#include <atomic>

#include "blocks_common.cuh"
#include "gemm_internal.h"

namespace bvml {
namespace blocks {
namespace {

// The pairs of SMs that the plans count on (B200: 148 SMs). A constant, so that
// a workspace's size needs no device; the launch takes the device's own count.
constexpr int kPairs = 74;

constexpr uint32_t kWaitLimit = 1u << 22;
std::atomic<uint32_t> g_wait_limit{kWaitLimit};

// An operand as stored: rows x cols, cols contiguous.
struct Stored {
    const void* p;
    long long ld;
    int rows, cols;
    bool pack;         // its rows do not start on 16 bytes: copied to the workspace
    size_t at;         // ... there
    long long ld_packed;
};

// A matrix of the epilogue whose rows do not start on 16 bytes (or, for outputs, end
// there), or a vector that does not: it lives in the workspace, on whole lines, while the
// kernel runs. (57600 x 128 -> 576 with a bias off 16 bytes: 24 us; read in place, one element
// after the other, 1266.)
struct Moved {
    bool on;
    size_t at;
    long long ld;
};

struct Plan {
    bool skinny;
    int bn;        // tile: columns of a pair
    int tok;       // skinny: tokens of a CTA
    int splits;    // shares of K
    int steps[2];
    int tiles_m, tiles_n;
    Stored a[2], b[2];
    Moved residual, out[2], save[2];
    Moved vectors[3];  // bias, col_scale
    long long ldslab;
    size_t slab;   // offset of the partial sums
    size_t bytes;  // workspace
};

int cdiv(int a, int b) { return (int)(((long long)a + b - 1) / b); }

// A product's cost in K steps of a 256-column tile (512 cycles, 0.3 us): the turns
// that the pairs take, times the longer of a tile's K steps and its epilogue. Both were
// measured: a step takes as long as its operands take to arrive, (128 + bn / 2) rows a
// CTA, whatever the tensor cores need for a narrower tile (8192 x 4096 x 8192: 310 us
// with 256 columns). An epilogue of scales and biases at most (`light`) takes 0.027 steps a
// column and 0.7 more a tile (57600 x 128 -> 1024: 32.8, 33.8, 34.4 and 38.4 us with 256,
// 192, 128 and 64 columns; -> 576: 25.9, 20.7, 23.7 and 23.8), any other twice that.
// Shares of K are written and read once more (6.5 TB/s), which fewer idle pairs have to
// earn back. Where it misses (us, its choice and the best): 57600 x 576 -> 128 18.9 and 16.7
// with 128 columns, 57600 x 64 -> 192 11.3 and 10.3 with 192, 57600 x 128 -> 1024 34.5 and
// 32.8 with 256.
double tile_cost(int tiles, int steps, int splits, int bn, double outputs, bool light) {
    const double rate = (128 + bn / 2) / 256.0;
    const long long turns = ((long long)tiles * splits + kPairs - 1) / kPairs;
    const double main = rate * steps / splits;
    const double epilogue = light ? 0.027 * bn + 0.7 : 0.054 * bn + 1.0;
    const double join = splits > 1 ? 7.0 + outputs * (6.0 * splits + 2.0) / 6.5e6 / 0.3 : 0.0;
    return turns * (main > epilogue ? main : epilogue) + epilogue + join;
}

Plan plan_of(const GemmLaunch& L) {
    Plan p{};
    const bool f8 = L.in_type == BVML_E4M3;
    const size_t es = elem_size(L.in_type);
    const int step = f8 ? 128 : 64;
    const int segs = L.k[1] > 0 ? 2 : 1;
    for (int i = 0; i < 2; ++i) p.steps[i] = i < segs ? cdiv(L.k[i], step) : 0;
    const int steps = p.steps[0] + p.steps[1];

    // operands: A by segment, B by segment or gate and up
    size_t off = 0;
    auto stored = [&](const void* ptr, long long ld, int rows, int cols) {
        Stored s{ptr, ld, rows, cols};
        if (rows == 1) s.ld = cols;  // one row has no pitch
        // (one row's pitch is made up where the tensor map is)
        s.pack = rows == 1 ? (reinterpret_cast<uintptr_t>(ptr) & 15) != 0 : !on16(ptr, ld, es);
        // whole 128-byte lines: a K step of a row then lies in one
        s.ld_packed = ((long long)cols * (long long)es + 127) / 128 * 128 / (long long)es;
        if (s.pack) {
            s.at = off;
            off += round256((size_t)rows * s.ld_packed * es);
        }
        return s;
    };
    for (int i = 0; i < segs; ++i)
        p.a[i] = L.a_t ? stored(L.a[i], L.lda[i], L.k[i], L.M)
                       : stored(L.a[i], L.lda[i], L.M, L.k[i]);
    for (int i = 0; i < (L.gated ? 2 : segs); ++i) {
        const int k = L.gated ? L.k[0] : L.k[i];
        p.b[i] = L.b_t ? stored(L.b[i], L.ldb[i], k, L.N) : stored(L.b[i], L.ldb[i], L.N, k);
    }

    p.splits = 1;
    // Few rows: the kernel that streams the weights, up to 64 rows, and up to 128 where
    // the weights are many or gated. us, bf16, N x K, that kernel at 64 rows and the tiles at
    // 65: 512 x 512 6.5 and 5.5, 8192 x 1024 11.2 and 8.9, 1024 x 8192 11.2 and 11.9 (with bias
    // and residual, for which the tiles share out no K, 11.6 and 22.7); that kernel at 128 and
    // the tiles at 129: 4096 x 4096 17.1 and 19.6 (bias and residual 17.7 and 17.0; at 65 rows
    // that kernel takes 14.3), 11264 x 4096 27.1 and 26.9, gated 43.4 and 52.7.
    const bool many = L.gated || (double)L.N * L.k[0] * (double)es > 20e6;
    if (!L.a_t && !L.b_t && L.M <= (many ? 128 : 64)) {
        p.skinny = true;
        p.tok = L.M <= 16 ? 16 : L.M <= 32 ? 32 : L.M <= 64 ? 64 : 128;
        const int tiles = cdiv(L.N, L.gated ? 64 : 128);
        // up to what the SMs hold at once, and at least two K steps a CTA
        const int slots = 2 * kPairs * (p.tok <= 64 ? 3 : 2);
        while (p.splits < 8 && (long long)tiles * p.splits * 2 <= slots && steps >= 4 * p.splits)
            p.splits *= 2;
        p.bytes = off;
        return p;
    }
    p.tiles_m = cdiv(L.M, 256);
    // K is shared out only where nothing but the sum is wanted: long sums over few
    // output tiles
    const bool light = !L.gated && !L.residual && !L.save[0] && L.act == BVML_ACT_NONE;
    const bool plain = light && !L.bias && !L.row_scale;
    double best = 1e300;
    const bool halves = L.gated || L.b_t;  // 256 and 128 columns only
    for (int bn = 256; bn >= (halves ? 128 : 64); bn -= halves ? 128 : 64) {
        const int tn = cdiv(L.N, L.gated ? bn / 2 : bn);
        for (int sp = 1; sp <= (plain ? 32 : 1) && (sp == 1 || steps / sp >= 8); sp *= 2) {
            const double c = tile_cost(p.tiles_m * tn, steps, sp, bn, (double)L.M * L.N, light);
            if (c < best * 0.999) {
                best = c;
                p.bn = bn;
                p.splits = sp;
                p.tiles_n = tn;
            }
        }
    }
    p.slab = off;
    if (p.splits > 1) {
        p.ldslab = ((long long)L.N + 31) / 32 * 32;
        off += round256((size_t)p.splits * L.M * p.ldslab * 4);
    } else {
        const size_t eo = elem_size(L.out_type);
        const long long lines = ((long long)L.N * (long long)eo + 127) / 128 * 128 / (long long)eo;
        auto moved = [&](const void* ptr, long long ld, int rows, bool output) {
            Moved m{};
            m.on = ptr && (!on16(ptr, ld, eo) || (output && ((size_t)L.N * eo & 15)));
            m.ld = m.on ? lines : ld;
            m.at = off;
            if (m.on) off += round256((size_t)rows * lines * eo);
            return m;
        };
        const int rows = L.out2 ? L.rows0 : L.M;
        p.residual = moved(L.residual, L.ldr, L.M, false);
        p.out[0] = moved(L.out, L.ldo, rows, true);
        p.out[1] = moved(L.out2, L.ldo2, rows, true);
        for (int i = 0; i < 2; ++i) p.save[i] = moved(L.save[i], L.lds[i], L.M, true);
        const float* const vectors[3] = {L.bias, L.col_scale[0], L.col_scale[1]};
        for (int i = 0; i < 3; ++i) {
            p.vectors[i].on = (reinterpret_cast<uintptr_t>(vectors[i]) & 15) != 0;
            p.vectors[i].at = off;
            if (p.vectors[i].on) off += round256((size_t)L.N * 4);
        }
    }
    p.bytes = off;
    return p;
}

// ------------------------------------------------------- operands laid out anew

// Rows of `cols` elements to a pitch of 16-byte units, eight (16-bit) or sixteen
// (8-bit) elements a thread; what pads a row's last unit is zeros.
template <typename T>
__global__ void __launch_bounds__(256)
pack_kernel(const T* src, long long ld, int rows, int cols, T* dst,
            int units) {
    constexpr int kE = 16 / sizeof(T);
    const long long total = (long long)rows * units;
    begin();
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total;
         i += (long long)gridDim.x * 256) {
        const long long r = i / units;
        const int c = (int)(i - r * units) * kE;
        const T* s = src + r * ld + c;
        uint4 u = make_uint4(0, 0, 0, 0);
        T* e = reinterpret_cast<T*>(&u);
#pragma unroll
        for (int j = 0; j < kE; ++j)
            if (c + j < cols) e[j] = s[j];
        *reinterpret_cast<uint4*>(dst + i * kE) = u;
    }
}

cudaError_t pack_rows(const void* src, long long ld, int rows, int cols, void* dst,
                      long long ld_packed, size_t es, cudaStream_t st) {
    const int units = (int)(ld_packed * (long long)es / 16);
    const long long want = ((long long)rows * units + 255) / 256;
    const int grid = (int)(want < 148 * 16 ? want : 148 * 16);
    if (es == 1)
        return launch_pdl(pack_kernel<uint8_t>, grid, 256, 0, st, true,
                          static_cast<const uint8_t*>(src), ld, rows, cols,
                          static_cast<uint8_t*>(dst), units);
    if (es == 2)
        return launch_pdl(pack_kernel<uint16_t>, grid, 256, 0, st, true,
                          static_cast<const uint16_t*>(src), ld, rows, cols,
                          static_cast<uint16_t*>(dst), units);
    return launch_pdl(pack_kernel<uint32_t>, grid, 256, 0, st, true,
                      static_cast<const uint32_t*>(src), ld, rows, cols,
                      static_cast<uint32_t*>(dst), units);
}
cudaError_t pack(const Stored& s, size_t es, void* ws, cudaStream_t st) {
    return pack_rows(s.p, s.ld, s.rows, s.cols, static_cast<char*>(ws) + s.at, s.ld_packed, es, st);
}

// The way back: neighbouring lanes write neighbouring elements.
template <typename T>
__global__ void __launch_bounds__(256)
unpack_kernel(const T* src, long long lds, int rows, int cols, T* dst,
              long long ld) {
    begin();
    for (int r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* a = src + r * lds;
        T* b = dst + r * ld;
#pragma unroll 4
        for (int c = threadIdx.x; c < cols; c += 256) b[c] = a[c];
    }
}
cudaError_t unpack(const Moved& m, const void* ws, void* dst, long long ld, int rows, int cols,
                   size_t es, cudaStream_t st) {
    const void* src = static_cast<const char*>(ws) + m.at;
    const int grid = rows < 148 * 32 ? rows : 148 * 32;
    if (es == 2)
        return launch_pdl(unpack_kernel<uint16_t>, grid, 256, 0, st, true,
                          static_cast<const uint16_t*>(src), m.ld, rows, cols,
                          static_cast<uint16_t*>(dst), ld);
    return launch_pdl(unpack_kernel<uint32_t>, grid, 256, 0, st, true,
                      static_cast<const uint32_t*>(src), m.ld, rows, cols,
                      static_cast<uint32_t*>(dst), ld);
}

// ------------------------------------------------------------ the shares' sum

template <typename T>
__global__ void __launch_bounds__(256)
join_kernel(const float* slab, long long stride, long long lds, int splits, int N,
            T* out, long long ldo, T* out2, long long ldo2, int rows0,
            int rows1, bool vec) {
    const long long m = blockIdx.x;
    begin();
    T* o;
    if (!out2 || m < rows0) o = out + m * ldo;
    else if (m >= rows1) o = out2 + (m - rows1) * ldo2;
    else return;
    for (int n = (blockIdx.y * 256 + threadIdx.x) * 8; n < N; n += gridDim.y * 256 * 8) {
        float v[8], t[8];
        load8(slab + m * lds + n, v);
        for (int s = 1; s < splits; ++s) {
            load8(slab + s * stride + m * lds + n, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += t[e];
        }
        if (vec && n + 8 <= N) {
            store8(o + n, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (n + e < N) o[n + e] = from_f<T>(v[e]);
        }
    }
}

template <typename T>
cudaError_t join(const GemmLaunch& L, const Plan& p, const float* slab, bool vec, cudaStream_t s) {
    const dim3 grid((unsigned)L.M, (unsigned)cdiv(L.N, 256 * 8));
    return launch_pdl(join_kernel<T>, grid, 256, 0, s, true, slab, (long long)L.M * p.ldslab,
                      p.ldslab, p.splits, L.N, static_cast<T*>(L.out), L.ldo,
                      static_cast<T*>(L.out2), L.ldo2, L.rows0, L.rows1, vec);
}

// ------------------------------------------------------------------ tensor maps

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> cached{nullptr};
    PFN_cuTensorMapEncodeTiled_v12000 fn = cached.load(std::memory_order_acquire);
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) ==
                cudaSuccess &&
            q == cudaDriverEntryPointSuccess) {
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
            cached.store(fn, std::memory_order_release);
        }
    }
    return fn;
}

// Boxes of 128 bytes x box_rows in the 128-byte swizzle; what lies outside the
// matrix reads zeros, and is not written.
cudaError_t encode_rows(CUtensorMap* m, const void* base, long long ld, int rows, int cols,
                        int type, int box_rows) {
    PFN_cuTensorMapEncodeTiled_v12000 fn = encoder();
    if (!fn) return cudaErrorNotSupported;
    const size_t es = elem_size(type);
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld * es};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / es), (cuuint32_t)box_rows};
    const cuuint32_t es1[2] = {1, 1};
    const CUtensorMapDataType dt = type == BVML_E4M3   ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : type == BVML_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                   : type == BVML_F16  ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_FLOAT32;
    return fn(m, dt, 2, const_cast<void*>(base), dims, strides, box, es1,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? cudaSuccess
               : cudaErrorInvalidValue;
}
cudaError_t encode(CUtensorMap* m, const Stored& s, const void* ws, int type, int box_rows) {
    return encode_rows(m, s.pack ? static_cast<const char*>(ws) + s.at : s.p,
                       s.pack || s.rows == 1 ? s.ld_packed : s.ld, s.rows, s.cols, type, box_rows);
}

// MMA instruction descriptor: fp32 D; A and B bf16 (1), f16 or e4m3 (0);
// transpose bits; N / 8 and M / 16.
uint32_t idesc_of(int type, bool a_t, bool b_t, int M, int N) {
    const uint32_t f = type == BVML_BF16 ? 1 : 0;
    return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)a_t << 15) | ((uint32_t)b_t << 16) |
           ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

}  // namespace

size_t gemm_workspace_bytes(const GemmLaunch& L) {
    if (L.M == 0 || L.N == 0 || L.k[0] == 0) return 0;
    return plan_of(L).bytes;
}

cudaError_t launch_gemm(const GemmLaunch& L, void* ws, cudaStream_t s) {
    if (L.M == 0 || L.N == 0) return cudaSuccess;
    const Plan p = plan_of(L);
    const size_t es = elem_size(L.in_type), eo = elem_size(L.out_type);
    const int segs = p.steps[1] > 0 ? 2 : 1, nb = L.gated ? 2 : segs;
    cudaError_t e = cudaSuccess;
    TileMaps maps{};
    const int rows_b = p.skinny ? (L.gated ? 64 : 128) : p.bn / 2;
    for (int i = 0; i < segs && e == cudaSuccess; ++i) {
        if (p.a[i].pack) e = pack(p.a[i], es, ws, s);
        if (e == cudaSuccess)
            e = encode(&maps.a[i], p.a[i], ws, L.in_type,
                       L.a_t ? 64 : p.skinny ? p.tok : 128);
    }
    for (int i = 0; i < nb && e == cudaSuccess; ++i) {
        if (p.b[i].pack) e = pack(p.b[i], es, ws, s);
        if (e == cudaSuccess)
            e = encode(&maps.b[i], p.b[i], ws, L.in_type, L.b_t ? 64 : rows_b);
    }
    if (e != cudaSuccess) return e;
    SkinnyArgs k{};
    TileArgs& a = k.t;
    a.M = L.M, a.N = L.N;
    a.steps[0] = p.steps[0], a.steps[1] = p.steps[1];
    a.tiles_m = p.tiles_m, a.tiles_n = p.tiles_n;
    a.splits = p.splits;
    a.row_scale = L.row_scale;
    for (int i = 0; i < 2; ++i) a.col_scale[i] = L.col_scale[i];
    a.bias = L.bias;
    a.rows0 = L.rows0, a.rows1 = L.rows1;
    a.out_rows = L.out2 ? L.rows0 : L.M;
    a.out_type = L.out_type, a.act = L.act;
    a.wait_limit = g_wait_limit.load(std::memory_order_relaxed);
    // the epilogue's matrices, or their places in the workspace
    auto place = [&](const Moved& m, const void* ptr) {
        return m.on ? static_cast<char*>(ws) + m.at : static_cast<char*>(const_cast<void*>(ptr));
    };
    auto pitch = [&](const Moved& m, long long ld) { return m.on ? m.ld : ld; };
    if (p.residual.on)
        e = pack_rows(L.residual, L.ldr, L.M, L.N, place(p.residual, nullptr), p.residual.ld, eo, s);
    if (e != cudaSuccess) return e;
    a.residual = place(p.residual, L.residual), a.ldr = pitch(p.residual, L.ldr);
    a.out = place(p.out[0], L.out), a.ldo = pitch(p.out[0], L.ldo);
    a.out2 = place(p.out[1], L.out2), a.ldo2 = pitch(p.out[1], L.ldo2);
    for (int i = 0; i < 2; ++i) {
        a.save[i] = place(p.save[i], L.save[i]);
        a.lds[i] = pitch(p.save[i], L.lds[i]);
    }
    // what the addresses and pitches that the epilogue touches have in common
    auto bits = [&](const void* ptr, long long ld) {
        return ptr ? reinterpret_cast<uintptr_t>(ptr) | (uintptr_t)ld * eo : (uintptr_t)0;
    };
    const uintptr_t out = bits(a.out, a.ldo) | bits(a.out2, a.ldo2);
    const uintptr_t save = bits(a.save[0], a.lds[0]) | bits(a.save[1], a.lds[1]);
    const uintptr_t all = out | save | bits(a.residual, a.ldr) |
                          reinterpret_cast<uintptr_t>(L.bias) |
                          reinterpret_cast<uintptr_t>(L.col_scale[0]) |
                          reinterpret_cast<uintptr_t>(L.col_scale[1]);
    a.vec = ((all & 15) == 0 ? kOn16 : 0) | ((save & 31) == 0 ? kWideSave : 0);
    if (p.skinny) {
        k.split = p.splits;
        a.idesc = idesc_of(L.in_type, false, false, 128, p.tok);
        return launch_skinny(p.tok, L.in_type == BVML_E4M3, L.gated, maps, k, s);
    }
    const float** const vectors[3] = {&a.bias, &a.col_scale[0], &a.col_scale[1]};
    for (int i = 0; i < 3; ++i) {
        if (!p.vectors[i].on) continue;
        float* to = reinterpret_cast<float*>(static_cast<char*>(ws) + p.vectors[i].at);
        e = pack_rows(*vectors[i], L.N, 1, L.N, to, (L.N + 3LL) / 4 * 4, 4, s);
        if (e != cudaSuccess) return e;
        *vectors[i] = to;
    }
    a.idesc = idesc_of(L.in_type, L.a_t, L.b_t, 256, p.bn);
    if (p.splits == 1) {  // one row's pitch is any multiple of 16 bytes
        auto tma = [&](long long ld) { return a.out_rows > 1 ? ld : (L.N + 7LL) / 8 * 8; };
        e = encode_rows(&maps.o[0], a.out, tma(a.ldo), a.out_rows, L.N, L.out_type, 32);
        if (e == cudaSuccess && a.out2)
            e = encode_rows(&maps.o[1], a.out2, tma(a.ldo2), a.out_rows, L.N, L.out_type, 32);
        if (e != cudaSuccess) return e;
    }
    if (p.splits > 1) {
        a.slab = reinterpret_cast<float*>(static_cast<char*>(ws) + p.slab);
        a.ldslab = p.ldslab;
    }
    a.by_tiles = divide_by((uint32_t)(p.tiles_m * p.tiles_n));
    // as many tile rows together as keep their rows of A at home in L2 (40 MB of 126:
    // the rest is for B passing through and the outputs), 4 to 64
    const long long row = 256LL * (p.steps[0] + p.steps[1]) * 128;
    a.group = 2;
    while (a.group < 6 && (row << (a.group + 1)) <= (40LL << 20)) ++a.group;
    a.by_group = divide_by((uint32_t)(p.tiles_n << a.group));
    int sms = 0;
    if ((e = sm_count(&sms)) != cudaSuccess) return e;
    const long long works = (long long)p.tiles_m * p.tiles_n * p.splits;
    const int pairs = (int)(works < sms / 2 ? works : sms / 2);
    if (L.b_t) e = launch_tile_grad(p.bn, L.a_t, maps, a, pairs, s);
    else if (L.in_type == BVML_E4M3) e = launch_tile_nt_f8(p.bn, L.gated, maps, a, pairs, s);
    else e = launch_tile_nt(p.bn, L.gated, maps, a, pairs, s);
    if (e != cudaSuccess) return e;
    if (p.splits == 1) {
        void* const to[4] = {L.out, L.out2, L.save[0], L.save[1]};
        const Moved* const from[4] = {&p.out[0], &p.out[1], &p.save[0], &p.save[1]};
        const long long ld[4] = {L.ldo, L.ldo2, L.lds[0], L.lds[1]};
        for (int i = 0; i < 4 && e == cudaSuccess; ++i)
            if (from[i]->on)
                e = unpack(*from[i], ws, to[i], ld[i], i < 2 ? a.out_rows : L.M, L.N, eo, s);
        return e;
    }
    const bool vec = on16(L.out, L.ldo, eo) && (!L.out2 || on16(L.out2, L.ldo2, eo));
    if (L.out_type == BVML_F16) return join<__half>(L, p, a.slab, vec, s);
    if (L.out_type == BVML_BF16) return join<__nv_bfloat16>(L, p, a.slab, vec, s);
    return join<float>(L, p, a.slab, vec, s);
}

uint32_t gemm_wait_limit(uint32_t attempts) { return g_wait_limit.exchange(attempts); }

cudaError_t gemm_errors(int* word) {
    *word = 0;
    cudaError_t (*readers[])(int*) = {tile_nt_error, tile_nt_f8_error, tile_grad_error,
                                      skinny_error};
    for (auto r : readers) {
        int w = 0;
        const cudaError_t e = r(&w);
        if (e != cudaSuccess) return e;
        if (w) *word = w;
    }
    return cudaSuccess;
}

}  // namespace blocks
}  // namespace bvml
