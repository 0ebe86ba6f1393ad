// extern "C" entry points of libbvml_blocks.so (declared in
// include/bvml_blocks.h): argument checks, workspace layout and the order of
// launches. Nothing here allocates or throws; the last failure's text is kept
// in a fixed buffer of the calling thread.
#include "blocks_internal.h"
#include "../trace.h"

#include <cstdarg>
#include <cstdio>

namespace {

using namespace bvml::blocks;

thread_local char g_error[512];

int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(g_error, sizeof(g_error), fmt, ap);
    va_end(ap);
    return code;
}
// A failed runtime call also sets the thread's last-error state: read and
// reset it, so that the next call's launch checks do not report it again.
int finish(cudaError_t e, const char* op) {
    if (e == cudaSuccess) {
        g_error[0] = 0;
        return BVML_OK;
    }
    (void)cudaGetLastError();
    return fail(BVML_ECUDA, "dsine cuda: %s: %s", op, cudaGetErrorString(e));
}
int einval(const char* op, const char* what) {
    return fail(BVML_EINVAL, "dsine ops: %s: %s", op, what);
}

// A matrix argument as the checks see it.
struct Mat {
    const void* p;
    long long ld;
    int rows, cols;
    size_t es;
    const char* name;
};

// nullptr if the matrix can be used, else what is wrong with it. An empty one
// may be null.
const char* mat_error(const Mat& m, char* buf, size_t n) {
    if (m.rows == 0) return nullptr;
    const char* why = nullptr;
    if (!m.p) why = "is null";
    else if (reinterpret_cast<uintptr_t>(m.p) % m.es) why = "is not aligned to its element type";
    else if (m.ld < m.cols && m.rows > 1) why = "has a row stride below its columns";
    else if (m.ld < 0 || m.ld > (1LL << 36)) why = "has a bad row stride";
    if (!why) return nullptr;
    std::snprintf(buf, n, "%s %s", m.name, why);
    return buf;
}

// Whether two matrices share a byte. Rows of one pitch that interleave (two
// column ranges of one buffer) do not.
bool overlap(const Mat& a, const Mat& b) {
    if (!a.p || !b.p || !a.rows || !b.rows || !a.cols || !b.cols) return false;
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
    const uintptr_t wa = (uintptr_t)a.cols * a.es, wb = (uintptr_t)b.cols * b.es;
    const uintptr_t sa = (uintptr_t)a.ld * a.es, sb = (uintptr_t)b.ld * b.es;
    const uintptr_t ea = pa + (a.rows - 1) * sa + wa, eb = pb + (b.rows - 1) * sb + wb;
    if (ea <= pb || eb <= pa) return false;
    if (sa != sb || sa == 0) return true;
    const uintptr_t d = pb >= pa ? (pb - pa) % sa : (sa - (pa - pb) % sa) % sa;
    return d < wa || d + wb > sa;
}

// Checks inputs and outputs; outputs may not overlap anything.
int check_mats(const char* op, const Mat* in, int n_in, const Mat* out, int n_out) {
    char buf[160];
    for (int i = 0; i < n_in; ++i)
        if (const char* e = mat_error(in[i], buf, sizeof(buf))) return einval(op, e);
    for (int i = 0; i < n_out; ++i) {
        if (const char* e = mat_error(out[i], buf, sizeof(buf))) return einval(op, e);
        for (int j = 0; j < n_in; ++j)
            if (overlap(out[i], in[j])) {
                std::snprintf(buf, sizeof(buf), "%s overlaps %s", out[i].name, in[j].name);
                return einval(op, buf);
            }
        for (int j = 0; j < i; ++j)
            if (overlap(out[i], out[j])) {
                std::snprintf(buf, sizeof(buf), "%s overlaps %s", out[i].name, out[j].name);
                return einval(op, buf);
            }
    }
    return BVML_OK;
}

// A list of matrices without an allocation; absent optional ones are left out.
struct Mats {
    Mat v[12];
    int n = 0;
    void add(const char* name, const void* p, long long ld, int rows, int cols, size_t es) {
        v[n++] = Mat{p, ld, rows, cols, es, name};
    }
    void opt(const char* name, const void* p, long long ld, int rows, int cols, size_t es) {
        if (p) add(name, p, ld, rows, cols, es);
    }
};

int check_workspace(const char* op, const void* ws, size_t have, size_t need) {
    if (need == 0) return BVML_OK;
    if (!ws || have < need)
        return fail(BVML_EWORKSPACE, "dsine ops: %s: workspace too small (%zu bytes needed)", op,
                    need);
    if (reinterpret_cast<uintptr_t>(ws) & 255)
        return fail(BVML_EWORKSPACE, "dsine ops: %s: workspace must be 256-byte aligned", op);
    return BVML_OK;
}

// The kernels' indexes are 32 bits past the last tile, their count of tiles too.
// (2^44 elements are 32 TB: no matrix that exists is refused by the product.)
constexpr int kMostRows = (1 << 30) - 64;
bool shape_ok(int T, int K, int N = 1) {
    auto size = [](int a, int b) { return (long long)a * b <= 1LL << 44; };
    return T >= 0 && K >= 1 && N >= 1 && T <= kMostRows && K <= kMostRows && N <= kMostRows &&
           size(T, K) && size(T, N) && size(N, K);
}

bool type16(int t) { return t == BVML_F16 || t == BVML_BF16; }
bool act_ok(int act) { return act >= BVML_ACT_NONE && act <= BVML_ACT_GELU; }

void* at(void* base, size_t off) { return static_cast<char*>(base) + off; }

// ---------------------------------------------------------------------- norm

int norm_entry(const char* op, const void* x, long long ldx, const void* r, long long ldr,
               const void* w, int T, int K, int type, int wtype, float eps, void* y,
               long long ldy, float* scale, bool quant, void* sum, long long lds, void* stream) {
    if (type != BVML_F32 && !type16(type)) return einval(op, "rows must be fp32, fp16 or bf16");
    if (wtype != BVML_F32 && wtype != type)
        return einval(op, "weights must be fp32 or of the rows' type");
    if (!shape_ok(T, K)) return einval(op, "bad shape");
    if (!(eps >= 0.0f)) return einval(op, "eps must not be negative");
    if (!w) return einval(op, "weight is null");
    if (sum && !r) return einval(op, "the sum is an output of the residual's addition");
    if (quant && !scale && T > 0) return einval(op, "scale is null");
    const size_t es = elem_size(type);
    Mats in, out;
    in.add("x", x, ldx, T, K, es);
    in.opt("residual", r, ldr, T, K, es);
    in.add("weight", w, K, 1, K, elem_size(wtype));
    out.add("y", y, ldy, T, K, quant ? 1 : es);
    out.opt("sum", sum, lds, T, K, es);
    if (quant) out.add("scale", scale, 1, T > 0 ? 1 : 0, T, 4);
    if (int e = check_mats(op, in.v, in.n, out.v, out.n)) return e;
    NormLaunch L{x, r, w, y, sum, quant ? scale : nullptr, ldx, ldr, ldy, lds, T, K, type, wtype, eps};
    return finish(launch_rms_norm(L, static_cast<cudaStream_t>(stream)), op);
}

size_t norm_backward_bytes(int T, int K) {
    return !shape_ok(T, K) ? 0 : round256((size_t)norm_backward_parts(T, K) * K * 4);
}

// ------------------------------------------------------------------ products

GemmLaunch linear_gemm(const bvml_linear_args& a) {
    GemmLaunch L{};
    L.a[0] = a.x, L.lda[0] = a.ldx;
    L.b[0] = a.w, L.ldb[0] = a.ldw;
    L.k[0] = a.K, L.M = a.T, L.N = a.N;
    L.in_type = a.in_type, L.out_type = a.out_type, L.act = a.act;
    L.row_scale = a.x_scale, L.col_scale[0] = a.w_scale;
    L.bias = a.bias, L.residual = a.residual, L.ldr = a.ldr;
    L.out = a.y, L.ldo = a.ldy;
    L.save[0] = a.z, L.lds[0] = a.ldz;
    return L;
}

GemmLaunch gated_gemm(const bvml_gated_args& a) {
    GemmLaunch L{};
    L.gated = true;
    L.a[0] = a.x, L.lda[0] = a.ldx;
    L.b[0] = a.w_gate, L.ldb[0] = a.ldw_gate;
    L.b[1] = a.w_up, L.ldb[1] = a.ldw_up;
    L.k[0] = a.K, L.M = a.T, L.N = a.F;
    L.in_type = a.in_type, L.out_type = a.out_type, L.act = a.act;
    L.row_scale = a.x_scale, L.col_scale[0] = a.gate_scale, L.col_scale[1] = a.up_scale;
    L.out = a.h, L.ldo = a.ldh;
    L.save[0] = a.g, L.lds[0] = a.ldg;
    L.save[1] = a.u, L.lds[1] = a.ldu;
    return L;
}

// dX (M, N) = dZ (M, k) W (k, N)
GemmLaunch grad_x_gemm(const void* dz, long long lddz, const void* w, long long ldw, int M, int N,
                       int k, int type, void* dx, long long lddx) {
    GemmLaunch L{};
    L.a[0] = dz, L.lda[0] = lddz;
    L.b[0] = w, L.ldb[0] = ldw, L.b_t = true;
    L.k[0] = k, L.M = M, L.N = N;
    L.in_type = L.out_type = type;
    L.out = dx, L.ldo = lddx;
    return L;
}

// dW (M, N) = dZ^T (M, k) X (k, N), dZ stored (k, M)
GemmLaunch grad_w_gemm(const void* dz, long long lddz, const void* x, long long ldx, int M, int N,
                       int k, int type, void* dw, long long lddw) {
    GemmLaunch L = grad_x_gemm(dz, lddz, x, ldx, M, N, k, type, dw, lddw);
    L.a_t = true;
    return L;
}

// An empty batch's row scales may be null, as its rows may.
const char* forward_types(int in_type, int out_type, int T, const void* xs, const void* ws0,
                          const void* ws1) {
    if (in_type == BVML_E4M3) {
        if ((!xs && T > 0) || !ws0 || !ws1) return "e4m3 inputs need their scales";
        if (!type16(out_type) && out_type != BVML_F32) return "output must be fp16, bf16 or fp32";
        return nullptr;
    }
    if (!type16(in_type)) return "inputs must be fp16, bf16 or e4m3";
    if (out_type != in_type && out_type != BVML_F32)
        return "output must be fp32 or of the inputs' type";
    return nullptr;
}

// 16-bit columns in whole 128-byte lines: a copy of the products' operands then
// touches one line a row and K step and not two.
long long whole_lines(int cols) { return ((long long)cols + 63) / 64 * 64; }

// linear_backward's workspace: dz (unless it is dy), the bias gradient's
// partial sums, the products' scratch.
struct LinearBackwardPlan {
    size_t dz = 0, partial = 0, gemm = 0, total = 0;
    long long lddz = 0;
    bool own_dz = false;
};
LinearBackwardPlan plan_of(const bvml_linear_backward_args& a, GemmLaunch* gx, GemmLaunch* gw,
                           void* ws) {
    LinearBackwardPlan p;
    p.own_dz = a.act != BVML_ACT_NONE;
    p.lddz = p.own_dz ? whole_lines(a.N) : a.lddy;
    const bool products = a.dx || a.dw;
    p.partial = p.own_dz && products ? round256((size_t)a.T * p.lddz * 2) : 0;
    p.gemm = p.partial + (a.dbias ? round256((size_t)act_backward_parts(a.T, a.N) * a.N * 4) : 0);
    // a place of the right alignment stands for the workspace where only its size is asked
    void* dz = p.own_dz ? (ws ? ws : reinterpret_cast<void*>(256)) : const_cast<void*>(a.dy);
    *gx = grad_x_gemm(dz, p.lddz, a.w, a.ldw, a.T, a.K, a.N, a.type, a.dx, a.lddx);
    *gw = grad_w_gemm(dz, p.lddz, a.x, a.ldx, a.N, a.K, a.T, a.type, a.dw, a.lddw);
    size_t m = 0;
    if (a.dx) m = gemm_workspace_bytes(*gx);
    if (a.dw) {
        const size_t n = gemm_workspace_bytes(*gw);
        m = n > m ? n : m;
    }
    p.total = p.gemm + m;
    return p;
}

// gated_linear_backward's: dg | du side by side, the products' scratch.
struct GatedBackwardPlan {
    size_t gemm = 0, total = 0;
    int fp = 0;  // columns of each half
};
GatedBackwardPlan plan_of(const bvml_gated_backward_args& a, GemmLaunch* gx, GemmLaunch* gw,
                          void* ws) {
    GatedBackwardPlan p;
    p.fp = (int)whole_lines(a.F);
    p.gemm = round256((size_t)a.T * 2 * p.fp * 2);
    void* d = ws ? ws : reinterpret_cast<void*>(256);
    void* du = at(d, (size_t)p.fp * 2);
    const long long ld = 2LL * p.fp;
    *gx = grad_x_gemm(d, ld, a.w_gate, a.ldw_gate, a.T, a.K, a.F, a.type, a.dx, a.lddx);
    gx->a[1] = du, gx->lda[1] = ld;
    gx->b[1] = a.w_up, gx->ldb[1] = a.ldw_up;
    gx->k[1] = a.F;
    *gw = grad_w_gemm(d, ld, a.x, a.ldx, p.fp + a.F, a.K, a.T, a.type, a.dw_gate, a.lddw_gate);
    gw->out2 = a.dw_up, gw->ldo2 = a.lddw_up;
    gw->rows0 = a.F, gw->rows1 = p.fp;
    size_t m = 0;
    if (a.dx) m = gemm_workspace_bytes(*gx);
    if (a.dw_gate) {
        const size_t n = gemm_workspace_bytes(*gw);
        m = n > m ? n : m;
    }
    p.total = p.gemm + m;
    return p;
}

cudaError_t zero_rows(void* p, long long ld, int rows, int cols, size_t es, cudaStream_t s) {
    return cudaMemset2DAsync(p, (size_t)(rows > 1 ? ld : cols) * es, 0, (size_t)cols * es, rows, s);
}

int check_linear(const bvml_linear_args* a) {
    const char* op = "linear";
    if (!a) return einval(op, "no arguments");
    if (!shape_ok(a->T, a->K, a->N)) return einval(op, "bad shape");
    if (const char* e =
            forward_types(a->in_type, a->out_type, a->T, a->x_scale, a->w_scale, a->w_scale))
        return einval(op, e);
    if (a->in_type != BVML_E4M3 && (a->x_scale || a->w_scale))
        return einval(op, "scales belong to e4m3 inputs");
    if (!act_ok(a->act)) return einval(op, "unknown activation");
    const size_t ei = elem_size(a->in_type), eo = elem_size(a->out_type);
    Mats in, out;
    in.add("x", a->x, a->ldx, a->T, a->K, ei);
    in.add("w", a->w, a->ldw, a->N, a->K, ei);
    if (a->T > 0) in.opt("x_scale", a->x_scale, a->T, 1, a->T, 4);
    in.opt("w_scale", a->w_scale, a->N, 1, a->N, 4);
    in.opt("bias", a->bias, a->N, 1, a->N, 4);
    in.opt("residual", a->residual, a->ldr, a->T, a->N, eo);
    out.add("y", a->y, a->ldy, a->T, a->N, eo);
    out.opt("z", a->z, a->ldz, a->T, a->N, eo);
    return check_mats(op, in.v, in.n, out.v, out.n);
}

int check_gated(const bvml_gated_args* a) {
    const char* op = "gated_linear";
    if (!a) return einval(op, "no arguments");
    if (!shape_ok(a->T, a->K, a->F)) return einval(op, "bad shape");
    if (const char* e =
            forward_types(a->in_type, a->out_type, a->T, a->x_scale, a->gate_scale, a->up_scale))
        return einval(op, e);
    if (a->in_type != BVML_E4M3 && (a->x_scale || a->gate_scale || a->up_scale))
        return einval(op, "scales belong to e4m3 inputs");
    if (!act_ok(a->act) || a->act == BVML_ACT_NONE) return einval(op, "unknown activation");
    if (!a->g != !a->u) return einval(op, "g and u are kept together");
    const size_t ei = elem_size(a->in_type), eo = elem_size(a->out_type);
    Mats in, out;
    in.add("x", a->x, a->ldx, a->T, a->K, ei);
    in.add("w_gate", a->w_gate, a->ldw_gate, a->F, a->K, ei);
    in.add("w_up", a->w_up, a->ldw_up, a->F, a->K, ei);
    if (a->T > 0) in.opt("x_scale", a->x_scale, a->T, 1, a->T, 4);
    in.opt("gate_scale", a->gate_scale, a->F, 1, a->F, 4);
    in.opt("up_scale", a->up_scale, a->F, 1, a->F, 4);
    out.add("h", a->h, a->ldh, a->T, a->F, eo);
    out.opt("g", a->g, a->ldg, a->T, a->F, eo);
    out.opt("u", a->u, a->ldu, a->T, a->F, eo);
    return check_mats(op, in.v, in.n, out.v, out.n);
}

int check_linear_backward(const bvml_linear_backward_args* a) {
    const char* op = "linear_backward";
    if (!a) return einval(op, "no arguments");
    if (!shape_ok(a->T, a->K, a->N)) return einval(op, "bad shape");
    if (!type16(a->type)) return einval(op, "matrices must be fp16 or bf16");
    if (!act_ok(a->act)) return einval(op, "unknown activation");
    if (a->act == BVML_ACT_NONE && a->z) return einval(op, "z belongs to an activation");
    Mats in, out;
    in.add("dy", a->dy, a->lddy, a->T, a->N, 2);
    if (a->act != BVML_ACT_NONE) in.add("z", a->z, a->ldz, a->T, a->N, 2);
    if (a->dw) in.add("x", a->x, a->ldx, a->T, a->K, 2);
    if (a->dx) in.add("w", a->w, a->ldw, a->N, a->K, 2);
    out.opt("dx", a->dx, a->lddx, a->T, a->K, 2);
    out.opt("dw", a->dw, a->lddw, a->N, a->K, 2);
    out.opt("dbias", a->dbias, a->N, 1, a->N, 4);
    return check_mats(op, in.v, in.n, out.v, out.n);
}

int check_gated_backward(const bvml_gated_backward_args* a) {
    const char* op = "gated_linear_backward";
    if (!a) return einval(op, "no arguments");
    if (!shape_ok(a->T, a->K, a->F)) return einval(op, "bad shape");
    if (!type16(a->type)) return einval(op, "matrices must be fp16 or bf16");
    if (!act_ok(a->act) || a->act == BVML_ACT_NONE) return einval(op, "unknown activation");
    if (!a->dw_gate != !a->dw_up) return einval(op, "dw_gate and dw_up are computed together");
    Mats in, out;
    in.add("dh", a->dh, a->lddh, a->T, a->F, 2);
    in.add("g", a->g, a->ldg, a->T, a->F, 2);
    in.add("u", a->u, a->ldu, a->T, a->F, 2);
    if (a->dw_gate) in.add("x", a->x, a->ldx, a->T, a->K, 2);
    if (a->dx) {
        in.add("w_gate", a->w_gate, a->ldw_gate, a->F, a->K, 2);
        in.add("w_up", a->w_up, a->ldw_up, a->F, a->K, 2);
    }
    out.opt("dx", a->dx, a->lddx, a->T, a->K, 2);
    out.opt("dw_gate", a->dw_gate, a->lddw_gate, a->F, a->K, 2);
    out.opt("dw_up", a->dw_up, a->lddw_up, a->F, a->K, 2);
    return check_mats(op, in.v, in.n, out.v, out.n);
}

}  // namespace

extern "C" {

const char* bvml_blocks_last_error(void) { return g_error; }
int bvml_blocks_version(void) { return BVML_BLOCKS_VERSION; }

int bvml_blocks_status(void* stream) {
    cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
    int word = 0;
    if (e == cudaSuccess) e = gemm_errors(&word);
    if (e != cudaSuccess) return finish(e, "blocks_status");
    if (word)
        return fail(BVML_ECUDA, "dsine cuda: blocks_status: a matrix product's pipeline gave up "
                                "(code %d)", word);
    return finish(cudaSuccess, "");
}

unsigned bvml_blocks_wait_limit(unsigned attempts) { return gemm_wait_limit(attempts); }

int bvml_rms_norm(const void* x, long long ldx, const void* residual, long long ldr,
                  const void* weight, int T, int K, int dtype, int weight_dtype, float eps,
                  void* y, long long ldy, void* sum, long long lds, void* stream) {
    bvml::NvtxRange nvtx("bvml_rms_norm");
    return norm_entry("rms_norm", x, ldx, residual, ldr, weight, T, K, dtype, weight_dtype, eps, y,
                      ldy, nullptr, false, sum, lds, stream);
}

int bvml_rms_norm_e4m3(const void* x, long long ldx, const void* residual, long long ldr,
                       const void* weight, int T, int K, int dtype, int weight_dtype, float eps,
                       void* q, long long ldq, float* scale, void* sum, long long lds,
                       void* stream) {
    bvml::NvtxRange nvtx("bvml_rms_norm_e4m3");
    return norm_entry("rms_norm_e4m3", x, ldx, residual, ldr, weight, T, K, dtype, weight_dtype,
                      eps, q, ldq, scale, true, sum, lds, stream);
}

size_t bvml_rms_norm_backward_workspace_bytes(int T, int K) { return norm_backward_bytes(T, K); }

int bvml_rms_norm_backward(const void* dy, long long lddy, const void* s, long long lds,
                           const void* weight, const void* dsum, long long ldds, int T, int K,
                           int dtype, int weight_dtype, float eps, void* dx, long long lddx,
                           void* dweight, void* workspace, size_t workspace_bytes, void* stream) {
    bvml::NvtxRange nvtx("bvml_rms_norm_backward");
    const char* op = "rms_norm_backward";
    if (dtype != BVML_F32 && !type16(dtype)) return einval(op, "rows must be fp32, fp16 or bf16");
    if (weight_dtype != BVML_F32 && weight_dtype != dtype)
        return einval(op, "weights must be fp32 or of the rows' type");
    if (!shape_ok(T, K)) return einval(op, "bad shape");
    if (!(eps >= 0.0f)) return einval(op, "eps must not be negative");
    const size_t es = elem_size(dtype), ew = elem_size(weight_dtype);
    Mats in, out;
    in.add("dy", dy, lddy, T, K, es);
    in.add("s", s, lds, T, K, es);
    in.add("weight", weight, K, 1, K, ew);
    in.opt("dsum", dsum, ldds, T, K, es);
    out.add("dx", dx, lddx, T, K, es);
    out.add("dweight", dweight, K, 1, K, ew);
    if (int e = check_mats(op, in.v, in.n, out.v, out.n)) return e;
    if (int e = check_workspace(op, workspace, workspace_bytes, norm_backward_bytes(T, K)))
        return e;
    NormBackwardLaunch L{dy, s, weight, dsum, dx, dweight, static_cast<float*>(workspace),
                         lddy, lds, ldds, lddx, T, K, dtype, weight_dtype, eps};
    return finish(launch_rms_norm_backward(L, static_cast<cudaStream_t>(stream)), op);
}

size_t bvml_linear_workspace_bytes(const bvml_linear_args* a) {
    return check_linear(a) ? 0 : gemm_workspace_bytes(linear_gemm(*a));
}

int bvml_linear(const bvml_linear_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    bvml::NvtxRange nvtx("bvml_linear");
    if (int e = check_linear(a)) return e;
    const GemmLaunch L = linear_gemm(*a);
    if (int e = check_workspace("linear", workspace, workspace_bytes, gemm_workspace_bytes(L)))
        return e;
    return finish(launch_gemm(L, workspace, static_cast<cudaStream_t>(stream)), "linear");
}

size_t bvml_gated_linear_workspace_bytes(const bvml_gated_args* a) {
    return check_gated(a) ? 0 : gemm_workspace_bytes(gated_gemm(*a));
}

int bvml_gated_linear(const bvml_gated_args* a, void* workspace, size_t workspace_bytes,
                      void* stream) {
    bvml::NvtxRange nvtx("bvml_gated_linear");
    if (int e = check_gated(a)) return e;
    const GemmLaunch L = gated_gemm(*a);
    if (int e = check_workspace("gated_linear", workspace, workspace_bytes,
                                gemm_workspace_bytes(L)))
        return e;
    return finish(launch_gemm(L, workspace, static_cast<cudaStream_t>(stream)), "gated_linear");
}

size_t bvml_linear_backward_workspace_bytes(const bvml_linear_backward_args* a) {
    if (check_linear_backward(a)) return 0;
    GemmLaunch gx, gw;
    return plan_of(*a, &gx, &gw, nullptr).total;
}

int bvml_linear_backward(const bvml_linear_backward_args* a, void* workspace,
                         size_t workspace_bytes, void* stream) {
    bvml::NvtxRange nvtx("bvml_linear_backward");
    const char* op = "linear_backward";
    if (int e = check_linear_backward(a)) return e;
    GemmLaunch gx, gw;
    const LinearBackwardPlan p = plan_of(*a, &gx, &gw, workspace);
    if (int e = check_workspace(op, workspace, workspace_bytes, p.total)) return e;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    const bool products = a->dx || a->dw;
    float* partial = a->dbias ? static_cast<float*>(at(workspace, p.partial)) : nullptr;
    if ((p.own_dz && products) || a->dbias) {
        ActBackwardLaunch L{a->dy, a->z, p.own_dz && products ? workspace : nullptr, partial,
                            a->lddy, a->ldz, p.lddz, a->T, a->N, a->type, a->act};
        e = launch_act_backward(L, s);
        if (e == cudaSuccess && a->dbias)
            e = launch_column_sum(partial, a->T ? act_backward_parts(a->T, a->N) : 0, a->N,
                                  a->dbias, BVML_F32, s);
    }
    if (e == cudaSuccess && a->dx) e = launch_gemm(gx, at(workspace, p.gemm), s);
    if (e == cudaSuccess && a->dw)
        e = a->T ? launch_gemm(gw, at(workspace, p.gemm), s)
                 : zero_rows(a->dw, a->lddw, a->N, a->K, 2, s);
    return finish(e, op);
}

size_t bvml_gated_linear_backward_workspace_bytes(const bvml_gated_backward_args* a) {
    if (check_gated_backward(a)) return 0;
    GemmLaunch gx, gw;
    return plan_of(*a, &gx, &gw, nullptr).total;
}

int bvml_gated_linear_backward(const bvml_gated_backward_args* a, void* workspace,
                               size_t workspace_bytes, void* stream) {
    bvml::NvtxRange nvtx("bvml_gated_linear_backward");
    const char* op = "gated_linear_backward";
    if (int e = check_gated_backward(a)) return e;
    GemmLaunch gx, gw;
    const GatedBackwardPlan p = plan_of(*a, &gx, &gw, workspace);
    if (int e = check_workspace(op, workspace, workspace_bytes, p.total)) return e;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    if (a->T == 0) {
        if (a->dw_gate) e = zero_rows(a->dw_gate, a->lddw_gate, a->F, a->K, 2, s);
        if (a->dw_gate && e == cudaSuccess)
            e = zero_rows(a->dw_up, a->lddw_up, a->F, a->K, 2, s);
        return finish(e, op);
    }
    GatedBackwardLaunch L{a->dh, a->g, a->u, workspace, at(workspace, (size_t)p.fp * 2),
                          a->lddh, a->ldg, a->ldu, 2LL * p.fp, a->T, a->F, a->type, a->act};
    if (a->dx || a->dw_gate) e = launch_gated_backward(L, s);
    if (e == cudaSuccess && a->dx) e = launch_gemm(gx, at(workspace, p.gemm), s);
    if (e == cudaSuccess && a->dw_gate) e = launch_gemm(gw, at(workspace, p.gemm), s);
    return finish(e, op);
}

}  // extern "C"
