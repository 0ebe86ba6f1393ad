// Python binding of the feed-forward operators: torch tensors in, torch tensors
// out, over the C ABI (include/bvml_blocks.h). Compiled into
// _lib/_blocks_torch.*.so (CPython and torch's C++ API): a call checks its
// tensors, allocates its outputs and launches in half the host time of the same
// steps in Python (one-token rms_norm with residual: 11.5 us a call there), which is
// what a decoding step with one-token operators is bound by.
//
// Arguments are positional; brovisionml_b200/blocks.py has the documented
// functions. Errors are RuntimeError("dsine ops: <op>: ...") as in the C ABI.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <optional>
#include <string>
#include <vector>

#include "bvml_blocks.h"

namespace {

using at::ScalarType;
using at::Tensor;

struct Refusal {
    std::string what;
};
struct Raised {};  // a Python exception is set already

// One call: its name, device, and the checks that every operator makes.
struct Call {
    const char* op;
    int dev = -1;

    [[noreturn]] void refuse(const std::string& what) const {
        throw Refusal{std::string("dsine ops: ") + op + ": " + what};
    }

    // Every given tensor on one CUDA device, and none that torch would follow past the
    // kernels: through autograd, forward-mode derivatives, a trace, a transform (vmap,
    // functionalize, ...) or a class of its own. These calls do not pass its dispatcher, so
    // that what it follows would be dropped, or held as a constant, without a word.
    void device(std::initializer_list<const Tensor*> ts) {
        using c10::DispatchKey;
        using Mode = c10::impl::TorchDispatchModeTLS;
        constexpr c10::DispatchKeySet kWrapped{
            DispatchKey::Python,      DispatchKey::Functionalize,
            DispatchKey::Batched,     DispatchKey::BatchedNestedTensor,
            DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper};
        const Tensor& first = **ts.begin();
        const c10::AutogradState& state = c10::AutogradState::get_tls_state();
        const bool grad = state.get_grad_mode(), forward = state.get_fw_grad_mode();
        if (at::tracer::impl::is_dispatch_enabled() ||
            (c10::impl::dispatch_mode_enabled() &&
             (Mode::get_mode(c10::impl::TorchDispatchModeKey::PROXY) ||
              Mode::get_mode(c10::impl::TorchDispatchModeKey::FAKE) ||
              Mode::get_mode(c10::impl::TorchDispatchModeKey::FUNCTIONAL))))
            refuse("cannot be traced");
        for (const Tensor* t : ts) {
            if (!t->defined()) continue;
            if (t->device() != first.device()) refuse("all inputs must share a device");
            if (grad && t->requires_grad())
                refuse("no autograd: pass detached tensors, or call under torch.no_grad() "
                       "(the gradients have functions of their own, *_backward)");
            if (forward && t->_fw_grad(0).defined())
                refuse("no forward-mode derivatives: pass tensors without a tangent");
            if (t->key_set().has_any(kWrapped))
                refuse("tensors of torch's transforms and of classes that torch dispatches "
                       "on are not followed: pass plain tensors");
            if (t->is_neg() || t->_is_zerotensor())
                refuse("a tensor's memory must hold its values: call resolve_neg() on a lazy "
                       "negation, clone() a zero tensor");
            if (t->layout() != at::kStrided) refuse("tensors must be strided");
        }
        if (!first.is_cuda())
            refuse("tensors must be CUDA-resident (this library has no CPU path)");
        dev = first.get_device();
    }

    int type(ScalarType t) const {
        switch (t) {
            case ScalarType::Float: return BVML_F32;
            case ScalarType::Half: return BVML_F16;
            case ScalarType::BFloat16: return BVML_BF16;
            case ScalarType::Float8_e4m3fn: return BVML_E4M3;
            default: refuse(std::string("unsupported storage dtype ") + c10::toString(t));
        }
    }
};

// A matrix: leading axes as rows, `ld` elements apart.
struct Rows {
    void* p = nullptr;
    long long ld = 0;
    int T = 0, K = 0;
};

Rows rows_of(const Call& c, const Tensor& t, const char* name) {
    const auto n = [&] { return std::string(name); };
    const int64_t d = t.dim();
    if (d == 0) c.refuse(n() + " must have rows of features");
    const auto size = t.sizes();
    const int64_t K = size[d - 1];
    int64_t T = 1;
    for (int64_t i = 0; i + 1 < d; ++i) T *= size[i];
    if (T > INT32_MAX || K > INT32_MAX) c.refuse(n() + " is too large");
    Rows r;
    r.T = (int)T;
    r.K = (int)K;
    r.ld = K;
    r.p = t.data_ptr();
    if (t.is_contiguous()) return r;
    const auto stride = t.strides();
    if (K > 1 && stride[d - 1] != 1) c.refuse(n() + "'s last axis must be contiguous");
    if (T <= 1) return r;
    int64_t ld = -1, span = 0;  // pitch, and elements that the axes so far cover
    for (int64_t i = d - 2; i >= 0; --i) {
        if (size[i] == 1) continue;
        if (ld < 0) ld = stride[i];
        else if (stride[i] != span) c.refuse(n() + "'s leading axes must be evenly spaced rows");
        span = stride[i] * size[i];
    }
    if (ld < K) c.refuse(n() + "'s rows overlap");
    r.ld = ld;
    return r;
}

Rows rows_of(const Call& c, const Tensor& t, const char* name, int cols, int rows,
             std::optional<ScalarType> type) {
    Rows r = rows_of(c, t, name);
    if (cols >= 0 && r.K != cols)
        c.refuse(std::string(name) + " has " + std::to_string(r.K) + " columns, expected " +
                 std::to_string(cols));
    if (rows >= 0 && r.T != rows)
        c.refuse(std::string(name) + " has " + std::to_string(r.T) + " rows, expected " +
                 std::to_string(rows));
    if (type && t.scalar_type() != *type)
        c.refuse(std::string(name) + " must be " + c10::toString(*type) + ", is " +
                 c10::toString(t.scalar_type()));
    return r;
}

// Pointer of a contiguous vector of n values, null for an absent one.
template <typename T = float>
const T* vec_of(const Call& c, const Tensor& t, const char* name, int64_t n,
                ScalarType type = ScalarType::Float) {
    if (!t.defined()) return nullptr;
    if (t.scalar_type() != type)
        c.refuse(std::string(name) + " must be " + c10::toString(type) + ", is " +
                 c10::toString(t.scalar_type()));
    if (t.numel() != n)
        c.refuse(std::string(name) + " has " + std::to_string(t.numel()) + " values, expected " +
                 std::to_string(n));
    if (!t.is_contiguous()) c.refuse(std::string(name) + " must be contiguous");
    return static_cast<const T*>(t.data_ptr());
}

Tensor make(at::IntArrayRef size, ScalarType type, int dev) {
    return Tensor(at::detail::empty_cuda(size, type, c10::Device(c10::kCUDA, (c10::DeviceIndex)dev),
                                         std::nullopt));
}
Tensor like(const Tensor& t, ScalarType type) { return make(t.sizes(), type, t.get_device()); }
// t's rows, `cols` columns
Tensor like(const Tensor& t, ScalarType type, int64_t cols) {
    c10::SmallVector<int64_t, 6> size(t.sizes().begin(), t.sizes().end());
    size.back() = cols;
    return make(size, type, t.get_device());
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

bool same_rows(const Tensor& a, const Tensor& b) {
    return a.dim() == b.dim() &&
           a.sizes().slice(0, a.dim() - 1) == b.sizes().slice(0, b.dim() - 1);
}

void check(int rc) {
    if (rc != BVML_OK) throw Refusal{bvml_blocks_last_error()};
}

// f(stream) with the call's device as the current one
template <typename F>
int on_device(const Call& c, F f) {
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != c.dev) guard.set_index((c10::DeviceIndex)c.dev);
    return f(static_cast<void*>(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)c.dev).stream()));
}

// An operator with a workspace: without one first, which most calls do not need.
template <typename A>
void run(const Call& c, int (*fn)(const A*, void*, size_t, void*), size_t (*bytes)(const A*),
         const A& a) {
    check(on_device(c, [&](void* stream) {
        const int rc = fn(&a, nullptr, 0, stream);
        if (rc != BVML_EWORKSPACE) return rc;
        const size_t need = bytes(&a);
        const Tensor ws = make({(int64_t)need}, ScalarType::Byte, c.dev);
        return fn(&a, ws.data_ptr(), need, stream);
    }));
}

// ------------------------------------------------------------------- arguments

Tensor tensor(PyObject* o, const char* name) {
    if (o == Py_None) return Tensor();
    if (!THPVariable_Check(o)) throw Refusal{std::string("dsine ops: ") + name + " must be a tensor"};
    return THPVariable_Unpack(o);
}
Tensor needed(PyObject* o, const char* name) {
    if (o == Py_None) throw Refusal{std::string("dsine ops: ") + name + " must be a tensor"};
    return tensor(o, name);
}
bool flag(PyObject* o) {  // read before anything else, as it may run Python code
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw Raised{};
    return v == 1;
}
std::optional<ScalarType> dtype(PyObject* o) {
    if (o == Py_None) return std::nullopt;
    if (!THPDtype_Check(o)) throw Refusal{"dsine ops: out_dtype must be a torch.dtype"};
    return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        throw Refusal{"dsine ops: eps must be a number"};
    }
    return v;
}

PyObject* out(const Tensor& t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}
PyObject* out(std::initializer_list<Tensor> ts) {
    PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
    if (!r) return nullptr;
    Py_ssize_t i = 0;
    for (const Tensor& t : ts) {
        PyObject* o = out(t);
        if (!o) {
            Py_DECREF(r);
            return nullptr;
        }
        PyTuple_SET_ITEM(r, i++, o);
    }
    return r;
}

// No C++ exception crosses into Python.
template <PyObject* (*F)(PyObject* const*)>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t) {
    try {
        return F(args);
    } catch (const Refusal& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what.c_str());
    } catch (const Raised&) {
    } catch (...) {  // torch's own: out of memory and the like
        torch::translate_exception_to_python(std::current_exception());
    }
    return nullptr;
}

// ------------------------------------------------------------------- operators

struct NormIn {
    Tensor x, w, r;
    Rows rx, rr;
    const void* pw;
    int type, wtype;
    float eps;
};
NormIn norm_in(Call& c, PyObject* const* a) {
    NormIn n;
    n.x = needed(a[0], "x");
    n.w = needed(a[1], "weight");
    n.r = tensor(a[2], "residual");
    n.eps = (float)number(a[3]);
    c.device({&n.x, &n.w, &n.r});
    n.rx = rows_of(c, n.x, "x");
    const ScalarType t = n.x.scalar_type(), wt = n.w.scalar_type();
    n.type = c.type(t);
    if (wt != t && wt != ScalarType::Float)
        c.refuse(std::string("weight must be Float or ") + c10::toString(t) + ", is " +
                 c10::toString(wt));
    n.wtype = c.type(wt);
    n.pw = vec_of<void>(c, n.w, "weight", n.rx.K, wt);
    if (n.r.defined()) {
        if (n.r.sizes() != n.x.sizes()) c.refuse("residual must have x's shape");
        n.rr = rows_of(c, n.r, "residual", n.rx.K, n.rx.T, t);
    }
    return n;
}

PyObject* rms_norm(PyObject* const* a) {
    Call c{"rms_norm"};
    const NormIn n = norm_in(c, a);
    const ScalarType t = n.x.scalar_type();
    const Tensor y = like(n.x, t), s = n.r.defined() ? like(n.x, t) : Tensor();
    check(on_device(c, [&](void* stream) {
        return bvml_rms_norm(n.rx.p, n.rx.ld, n.rr.p, n.rr.ld, n.pw, n.rx.T, n.rx.K, n.type,
                             n.wtype, n.eps, y.data_ptr(), n.rx.K, ptr(s), n.rx.K, stream);
    }));
    return s.defined() ? out({y, s}) : out(y);
}

PyObject* rms_norm_e4m3(PyObject* const* a) {
    Call c{"rms_norm_e4m3"};
    const NormIn n = norm_in(c, a);
    const Tensor q = like(n.x, ScalarType::Float8_e4m3fn);
    const Tensor scale = make(n.x.sizes().slice(0, n.x.dim() - 1), ScalarType::Float, c.dev);
    const Tensor s = n.r.defined() ? like(n.x, n.x.scalar_type()) : Tensor();
    check(on_device(c, [&](void* stream) {
        return bvml_rms_norm_e4m3(n.rx.p, n.rx.ld, n.rr.p, n.rr.ld, n.pw, n.rx.T, n.rx.K, n.type,
                                  n.wtype, n.eps, q.data_ptr(), n.rx.K,
                                  static_cast<float*>(scale.data_ptr()), ptr(s), n.rx.K, stream);
    }));
    return s.defined() ? out({q, scale, s}) : out({q, scale});
}

PyObject* rms_norm_backward(PyObject* const* a) {
    Call c{"rms_norm_backward"};
    const Tensor dy = needed(a[0], "dy"), s = needed(a[1], "s"), w = needed(a[2], "weight"),
                 ds = tensor(a[3], "dsum");
    const float eps = (float)number(a[4]);
    c.device({&dy, &s, &w, &ds});
    if (dy.sizes() != s.sizes() || (ds.defined() && ds.sizes() != s.sizes()))
        c.refuse("dy, s and dsum must have one shape");
    const ScalarType t = s.scalar_type(), wt = w.scalar_type();
    const Rows rs = rows_of(c, s, "s"), rd = rows_of(c, dy, "dy", rs.K, rs.T, t);
    const int type = c.type(t);
    if (wt != t && wt != ScalarType::Float)
        c.refuse(std::string("weight must be Float or ") + c10::toString(t) + ", is " +
                 c10::toString(wt));
    const void* pw = vec_of<void>(c, w, "weight", rs.K, wt);
    Rows re;
    if (ds.defined()) re = rows_of(c, ds, "dsum", rs.K, rs.T, t);
    const Tensor dx = like(s, t), dw = make({rs.K}, wt, c.dev);
    const size_t need = bvml_rms_norm_backward_workspace_bytes(rs.T, rs.K);
    check(on_device(c, [&](void* stream) {
        const Tensor ws = make({(int64_t)need}, ScalarType::Byte, c.dev);
        return bvml_rms_norm_backward(rd.p, rd.ld, rs.p, rs.ld, pw, re.p, re.ld, rs.T, rs.K, type,
                                      c.type(wt), eps, dx.data_ptr(), rs.K, dw.data_ptr(),
                                      ws.data_ptr(), need, stream);
    }));
    return out({dx, dw});
}

// The type of a product's output, and whether its scales are as its inputs want them.
ScalarType out_type(const Call& c, ScalarType in, std::optional<ScalarType> want,
                    std::initializer_list<const Tensor*> scales) {
    const bool e4m3 = in == ScalarType::Float8_e4m3fn;
    for (const Tensor* s : scales) {
        if (e4m3 && !s->defined()) c.refuse("e4m3 inputs need their scales");
        if (!e4m3 && s->defined()) c.refuse("scales belong to e4m3 inputs");
    }
    return want ? *want : e4m3 ? ScalarType::BFloat16 : in;
}

PyObject* linear(PyObject* const* a) {
    Call c{"linear"};
    const bool save = flag(a[8]);
    const Tensor x = needed(a[0], "x"), w = needed(a[1], "weight"), b = tensor(a[2], "bias"),
                 r = tensor(a[4], "residual"), xs = tensor(a[5], "x_scale"),
                 ws = tensor(a[6], "w_scale");
    c.device({&x, &w, &b, &r, &xs, &ws});
    const ScalarType t = x.scalar_type();
    const Rows rx = rows_of(c, x, "x"), rw = rows_of(c, w, "weight", rx.K, -1, t);
    const ScalarType o = out_type(c, t, dtype(a[7]), {&xs, &ws});
    bvml_linear_args g{};
    g.act = (int)PyLong_AsLong(a[3]);
    g.in_type = c.type(t);
    g.out_type = c.type(o);
    g.T = rx.T, g.K = rx.K, g.N = rw.T;
    g.x = rx.p, g.ldx = rx.ld;
    g.w = rw.p, g.ldw = rw.ld;
    g.x_scale = vec_of(c, xs, "x_scale", g.T);
    g.w_scale = vec_of(c, ws, "w_scale", g.N);
    g.bias = vec_of(c, b, "bias", g.N);
    if (r.defined()) {
        if (!same_rows(r, x)) c.refuse("residual must have the output's shape");
        const Rows rr = rows_of(c, r, "residual", g.N, g.T, o);
        g.residual = rr.p, g.ldr = rr.ld;
    }
    const Tensor y = like(x, o, g.N), z = save ? like(x, o, g.N) : Tensor();
    g.y = y.data_ptr(), g.z = ptr(z);
    g.ldy = g.ldz = g.N;
    run(c, bvml_linear, bvml_linear_workspace_bytes, g);
    return z.defined() ? out({y, z}) : out(y);
}

PyObject* linear_backward(PyObject* const* a) {
    Call c{"linear_backward"};
    const bool want_db = flag(a[5]), want_dx = flag(a[6]), want_dw = flag(a[7]);
    const Tensor dy = needed(a[0], "dy"), x = needed(a[1], "x"), w = needed(a[2], "weight"),
                 z = tensor(a[3], "z");
    c.device({&dy, &x, &w, &z});
    const ScalarType t = x.scalar_type();
    const Rows rx = rows_of(c, x, "x"), rw = rows_of(c, w, "weight", rx.K, -1, t);
    if (!same_rows(dy, x)) c.refuse("dy must have x's rows");
    bvml_linear_backward_args g{};
    g.act = (int)PyLong_AsLong(a[4]);
    g.type = c.type(t);
    g.T = rx.T, g.K = rx.K, g.N = rw.T;
    const Rows rd = rows_of(c, dy, "dy", g.N, g.T, t);
    if (z.defined() != (g.act != BVML_ACT_NONE))
        c.refuse("z belongs to an activation, and an activation needs it");
    if (z.defined()) {
        if (z.sizes() != dy.sizes()) c.refuse("z must have dy's shape");
        const Rows rz = rows_of(c, z, "z", g.N, g.T, t);
        g.z = rz.p, g.ldz = rz.ld;
    }
    g.dy = rd.p, g.lddy = rd.ld;
    g.x = rx.p, g.ldx = rx.ld;
    g.w = rw.p, g.ldw = rw.ld;
    const Tensor db = want_db ? make({g.N}, ScalarType::Float, c.dev) : Tensor();
    const Tensor dx = want_dx ? like(x, t) : Tensor();
    const Tensor dw = want_dw ? make({g.N, g.K}, t, c.dev) : Tensor();
    g.dx = ptr(dx), g.dw = ptr(dw), g.dbias = static_cast<float*>(ptr(db));
    g.lddx = g.lddw = g.K;
    run(c, bvml_linear_backward, bvml_linear_backward_workspace_bytes, g);
    return out({dx, dw, db});
}

PyObject* gated_linear(PyObject* const* a) {
    Call c{"gated_linear"};
    const bool save = flag(a[8]);
    const Tensor x = needed(a[0], "x"), wg = needed(a[1], "w_gate"), wu = needed(a[2], "w_up"),
                 xs = tensor(a[4], "x_scale"), gs = tensor(a[5], "gate_scale"),
                 us = tensor(a[6], "up_scale");
    c.device({&x, &wg, &wu, &xs, &gs, &us});
    const ScalarType t = x.scalar_type();
    const Rows rx = rows_of(c, x, "x"), rg = rows_of(c, wg, "w_gate", rx.K, -1, t),
               ru = rows_of(c, wu, "w_up", rx.K, rg.T, t);
    const ScalarType o = out_type(c, t, dtype(a[7]), {&xs, &gs, &us});
    bvml_gated_args g{};
    g.act = (int)PyLong_AsLong(a[3]);
    g.in_type = c.type(t);
    g.out_type = c.type(o);
    g.T = rx.T, g.K = rx.K, g.F = rg.T;
    g.x = rx.p, g.ldx = rx.ld;
    g.w_gate = rg.p, g.ldw_gate = rg.ld;
    g.w_up = ru.p, g.ldw_up = ru.ld;
    g.x_scale = vec_of(c, xs, "x_scale", g.T);
    g.gate_scale = vec_of(c, gs, "gate_scale", g.F);
    g.up_scale = vec_of(c, us, "up_scale", g.F);
    const Tensor h = like(x, o, g.F), pg = save ? like(x, o, g.F) : Tensor(),
                 pu = save ? like(x, o, g.F) : Tensor();
    g.h = h.data_ptr(), g.g = ptr(pg), g.u = ptr(pu);
    g.ldh = g.ldg = g.ldu = g.F;
    run(c, bvml_gated_linear, bvml_gated_linear_workspace_bytes, g);
    return save ? out({h, pg, pu}) : out(h);
}

PyObject* gated_linear_backward(PyObject* const* a) {
    Call c{"gated_linear_backward"};
    const bool want_dx = flag(a[7]), want_dw = flag(a[8]);
    const Tensor dh = needed(a[0], "dh"), x = needed(a[1], "x"), wg = needed(a[2], "w_gate"),
                 wu = needed(a[3], "w_up"), pg = needed(a[4], "g"), pu = needed(a[5], "u");
    c.device({&dh, &x, &wg, &wu, &pg, &pu});
    const ScalarType t = x.scalar_type();
    const Rows rx = rows_of(c, x, "x"), rg = rows_of(c, wg, "w_gate", rx.K, -1, t),
               ru = rows_of(c, wu, "w_up", rx.K, rg.T, t);
    if (!same_rows(dh, x) || pg.sizes() != dh.sizes() || pu.sizes() != dh.sizes())
        c.refuse("dh, g and u must have one shape, with x's rows");
    bvml_gated_backward_args g{};
    g.act = (int)PyLong_AsLong(a[6]);
    g.type = c.type(t);
    g.T = rx.T, g.K = rx.K, g.F = rg.T;
    const Rows rd = rows_of(c, dh, "dh", g.F, g.T, t), rpg = rows_of(c, pg, "g", g.F, g.T, t),
               rpu = rows_of(c, pu, "u", g.F, g.T, t);
    g.dh = rd.p, g.lddh = rd.ld;
    g.g = rpg.p, g.ldg = rpg.ld;
    g.u = rpu.p, g.ldu = rpu.ld;
    g.x = rx.p, g.ldx = rx.ld;
    g.w_gate = rg.p, g.ldw_gate = rg.ld;
    g.w_up = ru.p, g.ldw_up = ru.ld;
    const Tensor dx = want_dx ? like(x, t) : Tensor();
    const Tensor dg = want_dw ? make({g.F, g.K}, t, c.dev) : Tensor(),
                 du = want_dw ? make({g.F, g.K}, t, c.dev) : Tensor();
    g.dx = ptr(dx), g.dw_gate = ptr(dg), g.dw_up = ptr(du);
    g.lddx = g.lddw_gate = g.lddw_up = g.K;
    run(c, bvml_gated_linear_backward, bvml_gated_linear_backward_workspace_bytes, g);
    return out({dx, dg, du});
}

template <PyObject* (*F)(PyObject* const*), int N>
PyObject* counted(PyObject* self, PyObject* const* args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "%d arguments expected, %zd given", N, n);
        return nullptr;
    }
    return entry<F>(self, args, n);
}
#define BVML_METHOD(f, n) \
    {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(counted<f, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    BVML_METHOD(rms_norm, 4),      BVML_METHOD(rms_norm_e4m3, 4),
    BVML_METHOD(rms_norm_backward, 5), BVML_METHOD(linear, 9),
    BVML_METHOD(linear_backward, 8),   BVML_METHOD(gated_linear, 9),
    BVML_METHOD(gated_linear_backward, 9), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_blocks_torch", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__blocks_torch() { return PyModule_Create(&module); }
