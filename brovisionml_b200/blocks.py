"""Feed-forward operators over rows of features (pixels of a grid, tokens of a
sequence), the kernels of libbvml_blocks.so (include/bvml_blocks.h):

  rms_norm, rms_norm_e4m3   s = x + residual, s / sqrt(mean(s^2) + eps) * weight,
                            in the rows' type or in 8 bits with a scale a row
  linear                    act(x w^T + bias) + residual
  gated_linear              act(x w_gate^T) * (x w_up^T)

each with its backward pass as a function of its own (``*_backward``): the
operators take no part in torch's autograd, and refuse inputs that require
gradients while it records.

Matrices are 2-D, or have leading axes that are taken as rows; the last axis
is contiguous and rows may be further apart than they are long (a column range
of a wider tensor). fp16 and bf16, for the norm fp32 too; ``linear`` and
``gated_linear`` also take ``torch.float8_e4m3fn`` with fp32 scales, one a row
(``rms_norm_e4m3`` gives the rows, ``pack_weight_e4m3`` the weights). They run on the
tensors' device and its current torch stream, never synchronise, and
can be captured into a CUDA graph. There is no CPU path. Errors raise
``RuntimeError("dsine ops: ..." / "dsine cuda: ...")``.
"""
from __future__ import annotations

import ctypes
import os

import torch

from ._capi import BVML_F16, BVML_F32, BVML_OK, LIB_PATH

BLOCKS_LIB_PATH = os.path.join(os.path.dirname(LIB_PATH), "libbvml_blocks.so")
BVML_BF16 = 2
BVML_E4M3 = 3
BVML_EWORKSPACE = 4

# Every symbol include/bvml_blocks.h declares (checked by the CPU test suite).
EXPORTS = ("bvml_blocks_last_error", "bvml_blocks_version", "bvml_blocks_status",
           "bvml_rms_norm", "bvml_rms_norm_e4m3", "bvml_rms_norm_backward",
           "bvml_rms_norm_backward_workspace_bytes", "bvml_linear",
           "bvml_linear_workspace_bytes", "bvml_linear_backward",
           "bvml_linear_backward_workspace_bytes", "bvml_gated_linear",
           "bvml_gated_linear_workspace_bytes", "bvml_gated_linear_backward",
           "bvml_gated_linear_backward_workspace_bytes")

if not os.path.exists(BLOCKS_LIB_PATH):
    raise ImportError(
        f"brovisionml_b200: CUDA library not built ({BLOCKS_LIB_PATH} missing); run "
        "`python brovisionml_b200/build.py` (nvcc for sm_100a)")

blocks_lib = ctypes.CDLL(BLOCKS_LIB_PATH)

_vp, _i, _ll, _f, _sz = (ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float,
                         ctypes.c_size_t)


class LinearArgs(ctypes.Structure):
    """bvml_linear_args"""
    _fields_ = [(n, _vp) for n in ("x", "w", "x_scale", "w_scale", "bias", "residual", "y", "z")] \
        + [(n, _ll) for n in ("ldx", "ldw", "ldr", "ldy", "ldz")] \
        + [(n, _i) for n in ("T", "K", "N", "in_type", "out_type", "act")]


class LinearBackwardArgs(ctypes.Structure):
    """bvml_linear_backward_args"""
    _fields_ = [(n, _vp) for n in ("dy", "z", "x", "w", "dx", "dw", "dbias")] \
        + [(n, _ll) for n in ("lddy", "ldz", "ldx", "ldw", "lddx", "lddw")] \
        + [(n, _i) for n in ("T", "K", "N", "type", "act")]


class GatedArgs(ctypes.Structure):
    """bvml_gated_args"""
    _fields_ = [(n, _vp) for n in ("x", "w_gate", "w_up", "x_scale", "gate_scale", "up_scale",
                                   "h", "g", "u")] \
        + [(n, _ll) for n in ("ldx", "ldw_gate", "ldw_up", "ldh", "ldg", "ldu")] \
        + [(n, _i) for n in ("T", "K", "F", "in_type", "out_type", "act")]


class GatedBackwardArgs(ctypes.Structure):
    """bvml_gated_backward_args"""
    _fields_ = [(n, _vp) for n in ("dh", "g", "u", "x", "w_gate", "w_up", "dx", "dw_gate",
                                   "dw_up")] \
        + [(n, _ll) for n in ("lddh", "ldg", "ldu", "ldx", "ldw_gate", "ldw_up", "lddx",
                              "lddw_gate", "lddw_up")] \
        + [(n, _i) for n in ("T", "K", "F", "type", "act")]


def _bind(name, restype, argtypes):
    f = getattr(blocks_lib, name)
    f.restype, f.argtypes = restype, argtypes
    return f


_last_error = _bind("bvml_blocks_last_error", ctypes.c_char_p, [])
_bind("bvml_blocks_version", _i, [])
_status = _bind("bvml_blocks_status", _i, [_vp])
_norm = _bind("bvml_rms_norm", _i, [_vp, _ll, _vp, _ll, _vp, _i, _i, _i, _i, _f, _vp, _ll, _vp,
                                    _ll, _vp])
_norm_e4m3 = _bind("bvml_rms_norm_e4m3", _i, [_vp, _ll, _vp, _ll, _vp, _i, _i, _i, _i, _f, _vp,
                                              _ll, _vp, _vp, _ll, _vp])
_norm_bwd_ws = _bind("bvml_rms_norm_backward_workspace_bytes", _sz, [_i, _i])
_norm_bwd = _bind("bvml_rms_norm_backward", _i, [_vp, _ll, _vp, _ll, _vp, _vp, _ll, _i, _i, _i,
                                                 _i, _f, _vp, _ll, _vp, _vp, _sz, _vp])


def _bind_args(name, struct):
    p = ctypes.POINTER(struct)
    return (_bind(name, _i, [p, _vp, _sz, _vp]),
            _bind(name + "_workspace_bytes", _sz, [p]))


_linear, _linear_ws = _bind_args("bvml_linear", LinearArgs)
_linear_bwd, _linear_bwd_ws = _bind_args("bvml_linear_backward", LinearBackwardArgs)
_gated, _gated_ws = _bind_args("bvml_gated_linear", GatedArgs)
_gated_bwd, _gated_bwd_ws = _bind_args("bvml_gated_linear_backward", GatedBackwardArgs)

BLOCK_ACTIVATIONS = {"none": 0, "relu": 1, "sigmoid": 2, "tanh": 3, "silu": 4, "gelu": 5}
_E4M3 = torch.float8_e4m3fn
_TYPES = {torch.float32: BVML_F32, torch.float16: BVML_F16, torch.bfloat16: BVML_BF16,
          _E4M3: BVML_E4M3}
_F32 = torch.float32


def _err(op: str, what: str) -> RuntimeError:
    return RuntimeError(f"dsine ops: {op}: {what}")


def _check(rc: int) -> None:
    if rc != BVML_OK:
        msg = _last_error().decode("utf-8", "replace")
        raise RuntimeError(msg or f"dsine ops: failed with status {rc}")


def _device(op: str, *ts) -> int:
    """The index of the CUDA device that the tensors (or Nones) share."""
    dev = ts[0].get_device()
    grad = torch.is_grad_enabled()
    for t in ts:
        if t is None:
            continue
        if t.get_device() != dev:
            raise _err(op, "all inputs must share a device")
        if grad and t.requires_grad:
            raise _err(op, "no autograd: pass detached tensors, or call under torch.no_grad() "
                           "(the gradients have functions of their own, *_backward)")
    if dev < 0 or not ts[0].is_cuda:
        if any(t is not None and t.device != ts[0].device for t in ts):
            raise _err(op, "all inputs must share a device")
        raise _err(op, "tensors must be CUDA-resident (this library has no CPU path)")
    return dev


def _act(op: str, act: str) -> int:
    code = BLOCK_ACTIVATIONS.get(act)
    if code is None:
        raise _err(op, f"unknown activation {act!r}")
    return code


def _type(op: str, dt: torch.dtype) -> int:
    code = _TYPES.get(dt)
    if code is None:
        raise _err(op, f"unsupported storage dtype {dt}")
    return code


def _rows(op: str, t: torch.Tensor, name: str, cols: int | None = None, rows: int | None = None,
          dtype: torch.dtype | None = None):
    """(pointer, row stride, rows, columns) of a matrix."""
    shape = t.shape
    if len(shape) != 2:
        if len(shape) == 0:
            raise _err(op, f"{name} must have rows of features")
        if len(shape) == 1:
            t = t[None]
        else:
            n = 1
            for d in shape[:-1]:
                n *= d
            try:
                t = t.view(n, shape[-1])
            except RuntimeError:
                raise _err(op, f"{name}'s leading axes must be evenly spaced rows") from None
        shape = t.shape
    T, K = shape
    if cols is not None and K != cols:
        raise _err(op, f"{name} has {K} columns, expected {cols}")
    if rows is not None and T != rows:
        raise _err(op, f"{name} has {T} rows, expected {rows}")
    if dtype is not None and t.dtype != dtype:
        raise _err(op, f"{name} must be {dtype}, is {t.dtype}")
    if T > 0x7fffffff or K > 0x7fffffff:
        raise _err(op, f"{name} is too large")
    if t.is_contiguous():
        return t.data_ptr(), K, T, K
    s0, s1 = t.stride()
    if K > 1 and s1 != 1:
        raise _err(op, f"{name}'s last axis must be contiguous")
    if T > 1 and s0 < K:
        raise _err(op, f"{name}'s rows overlap")
    return t.data_ptr(), (s0 if T > 1 else K), T, K


def _vec(op: str, t: torch.Tensor | None, name: str, n: int, dtype: torch.dtype = _F32):
    """Pointer of a vector of n values, or None."""
    if t is None:
        return None
    if t.dtype != dtype:
        raise _err(op, f"{name} must be {dtype}, is {t.dtype}")
    if t.numel() != n:
        raise _err(op, f"{name} has {t.numel()} values, expected {n}")
    if not t.is_contiguous():
        raise _err(op, f"{name} must be contiguous")
    return t.data_ptr()


# The current stream's handle without a Stream object around it (2 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


_current_device = torch.cuda.current_device


def _call(dev: int, fn, *args) -> int:
    """fn(*args, stream) with `dev` as the current device and its current stream."""
    if _current_device() == dev:
        return fn(*args, _raw_stream(dev))
    with torch.cuda.device(dev):
        return fn(*args, _raw_stream(dev))


def _run(fn, ws_fn, args, dev: int) -> None:
    """fn(args), with a workspace only where the call without one is turned
    down (the common call needs none)."""
    p = ctypes.byref(args)
    rc = _call(dev, fn, p, None, 0)
    if rc == BVML_EWORKSPACE:
        need = ws_fn(p)
        ws = torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", dev))
        rc = _call(dev, fn, p, ws.data_ptr(), need)
    if rc:
        _check(rc)


def _like(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor like t."""
    return torch.empty_like(t) if t.is_contiguous() else \
        torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _new(t: torch.Tensor, cols: int, dtype: torch.dtype) -> torch.Tensor:
    """An uninitialised tensor of t's rows, `cols` columns."""
    return torch.empty((*t.shape[:-1], cols), dtype=dtype, device=t.device)


# ----------------------------------------------------------------------- norm


def _norm_inputs(op, x, weight, residual):
    dev = _device(op, x, weight, residual)
    px, ldx, T, K = _rows(op, x, "x")
    dt, wt = x.dtype, weight.dtype
    if wt != dt and wt != _F32:
        raise _err(op, f"weight must be float32 or {dt}, is {wt}")
    pw = _vec(op, weight, "weight", K, wt)
    pr, ldr = None, 0
    if residual is not None:
        if residual.shape != x.shape:
            raise _err(op, "residual must have x's shape")
        pr, ldr, _, _ = _rows(op, residual, "residual", K, T, dt)
    return dev, px, ldx, T, K, _type(op, dt), _TYPES[wt], pw, pr, ldr


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
             eps: float = 1e-6):
    """y = s / sqrt(mean(s^2) + eps) * weight with s = x + residual, row by row.
    x and residual (..., K) fp32, fp16 or bf16; weight (K) of that type or
    fp32. Returns y, or with a residual (y, s), both of x's type; the norm
    is taken of the unrounded sum."""
    dev, px, ldx, T, K, ty, wt, pw, pr, ldr = _norm_inputs("rms_norm", x, weight, residual)
    y = _like(x)
    if residual is None:
        rc = _call(dev, _norm, px, ldx, None, 0, pw, T, K, ty, wt, eps, y.data_ptr(), K, None, K)
        if rc:
            _check(rc)
        return y
    s = _like(x)
    rc = _call(dev, _norm, px, ldx, pr, ldr, pw, T, K, ty, wt, eps, y.data_ptr(), K, s.data_ptr(),
               K)
    if rc:
        _check(rc)
    return y, s


def rms_norm_e4m3(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
                  *, eps: float = 1e-6):
    """rms_norm with y in 8 bits, as ``linear`` and ``gated_linear`` take it:
    (q, scale) or, with a residual, (q, scale, s); q (..., K) float8_e4m3fn, scale (...)
    fp32, y ~ q * scale[..., None]. The row's largest magnitude becomes 448
    (scale 1 for a row of zeros; a row with NaN or infinities has a NaN scale)."""
    dev, px, ldx, T, K, ty, wt, pw, pr, ldr = _norm_inputs("rms_norm_e4m3", x, weight, residual)
    q = torch.empty(x.shape, dtype=_E4M3, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=_F32, device=x.device)
    s = _like(x) if residual is not None else None
    rc = _call(dev, _norm_e4m3, px, ldx, pr, ldr, pw, T, K, ty, wt, eps, q.data_ptr(), K,
               scale.data_ptr(), None if s is None else s.data_ptr(), K)
    if rc:
        _check(rc)
    return (q, scale) if s is None else (q, scale, s)


def rms_norm_backward(dy: torch.Tensor, s: torch.Tensor, weight: torch.Tensor,
                      dsum: torch.Tensor | None = None, *, eps: float = 1e-6):
    """(dx, dweight) of rms_norm: s is the sum its forward pass returned (x
    without a residual), dsum the gradient of that sum where it went on as
    the residual stream. dx is the gradient of x and of the residual alike."""
    op = "rms_norm_backward"
    dev = _device(op, dy, s, weight, dsum)
    if dy.shape != s.shape or dsum is not None and dsum.shape != s.shape:
        raise _err(op, "dy, s and dsum must have one shape")
    ps, lds, T, K = _rows(op, s, "s")
    dt, wt = s.dtype, weight.dtype
    pd, ldd, _, _ = _rows(op, dy, "dy", K, T, dt)
    if wt != dt and wt != _F32:
        raise _err(op, f"weight must be float32 or {dt}, is {wt}")
    pw = _vec(op, weight, "weight", K, wt)
    pr, ldr = None, 0
    if dsum is not None:
        pr, ldr, _, _ = _rows(op, dsum, "dsum", K, T, dt)
    ty = _type(op, dt)
    dx = _like(s)
    dw = torch.empty((K,), dtype=wt, device=s.device)
    need = _norm_bwd_ws(T, K)
    ws = torch.empty(need, dtype=torch.uint8, device=s.device)
    _check(_call(dev, _norm_bwd, pd, ldd, ps, lds, pw, pr, ldr, T, K, ty, _TYPES[wt], eps,
                 dx.data_ptr(), K, dw.data_ptr(), ws.data_ptr(), need))
    return dx, dw


# ------------------------------------------------------------------- products


def pack_weight_e4m3(weight: torch.Tensor):
    """(N, K) weights -> (q, scale) for ``linear`` / ``gated_linear``: e4m3 values
    and one fp32 scale an output feature, weight ~ q * scale[:, None]."""
    w = weight.detach().float()
    scale = w.abs().amax(1) / 448.0
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return (w / scale[:, None]).clamp(-448.0, 448.0).to(_E4M3), scale


def _out_type(op, in_dtype, out_dtype, scales):
    if in_dtype == _E4M3:
        if any(s is None for s in scales):
            raise _err(op, "e4m3 inputs need their scales")
        return torch.bfloat16 if out_dtype is None else out_dtype
    if any(s is not None for s in scales):
        raise _err(op, "scales belong to e4m3 inputs")
    return in_dtype if out_dtype is None else out_dtype


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
           act: str = "none", residual: torch.Tensor | None = None,
           x_scale: torch.Tensor | None = None, w_scale: torch.Tensor | None = None,
           out_dtype: torch.dtype | None = None, save: bool = False):
    """act(x weight^T + bias) + residual on the tensor cores, fp32 accumulation,
    one rounding. x (..., K), weight (N, K), bias (N) fp32, residual (..., N) of
    the output's type: the inputs' type or fp32 (``out_dtype``). e4m3 inputs come
    with x_scale (...) and w_scale (N), and give bf16 unless out_dtype says
    otherwise. act: none, relu, sigmoid, tanh, silu, gelu (erf form). Returns
    y (..., N), with save=True (y, z), z the pre-activation for linear_backward."""
    op = "linear"
    dev = _device(op, x, weight, bias, residual, x_scale, w_scale)
    px, ldx, T, K = _rows(op, x, "x")
    pw, ldw, N, _ = _rows(op, weight, "weight", K, None, x.dtype)
    od = _out_type(op, x.dtype, out_dtype, (x_scale, w_scale))
    ty, to = _type(op, x.dtype), _type(op, od)
    pr, ldr = None, 0
    if residual is not None:
        if residual.shape[:-1] != x.shape[:-1]:
            raise _err(op, "residual must have the output's shape")
        pr, ldr, _, _ = _rows(op, residual, "residual", N, T, od)
    y = _new(x, N, od)
    z = _new(x, N, od) if save else None
    a = LinearArgs(px, pw, _vec(op, x_scale, "x_scale", T), _vec(op, w_scale, "w_scale", N),
                   _vec(op, bias, "bias", N), pr, y.data_ptr(), None if z is None else z.data_ptr(),
                   ldx, ldw, ldr, N, N, T, K, N, ty, to, _act(op, act))
    _run(_linear, _linear_ws, a, dev)
    return (y, z) if save else y


def linear_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                    z: torch.Tensor | None = None, *, act: str = "none", bias: bool = False,
                    dx: bool = True, dw: bool = True):
    """(dx, dweight, dbias) of linear for fp16 or bf16 matrices: dy (..., N), x
    (..., K), weight (N, K), z (..., N) the pre-activation that linear(save=True)
    returned (None without an activation). dbias is fp32, None unless ``bias``; dx=False
    or dw=False leave that gradient out (None). The residual's gradient is dy."""
    op = "linear_backward"
    dev = _device(op, dy, x, weight, z)
    px, ldx, T, K = _rows(op, x, "x")
    pw, ldw, N, _ = _rows(op, weight, "weight", K, None, x.dtype)
    if dy.shape[:-1] != x.shape[:-1]:
        raise _err(op, "dy must have x's rows")
    pd, ldd, _, _ = _rows(op, dy, "dy", N, T, x.dtype)
    code, ty = _act(op, act), _type(op, x.dtype)
    pz, ldz = None, 0
    if (z is None) != (code == 0):
        raise _err(op, "z belongs to an activation, and an activation needs it")
    if z is not None:
        if z.shape != dy.shape:
            raise _err(op, "z must have dy's shape")
        pz, ldz, _, _ = _rows(op, z, "z", N, T, x.dtype)
    gx = _like(x) if dx else None
    gw = torch.empty((N, K), dtype=x.dtype, device=x.device) if dw else None
    gb = torch.empty((N,), dtype=_F32, device=x.device) if bias else None
    a = LinearBackwardArgs(pd, pz, px, pw, None if gx is None else gx.data_ptr(),
                           None if gw is None else gw.data_ptr(),
                           None if gb is None else gb.data_ptr(), ldd, ldz, ldx, ldw, K, K,
                           T, K, N, ty, code)
    _run(_linear_bwd, _linear_bwd_ws, a, dev)
    return gx, gw, gb


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, *,
                 act: str = "silu", x_scale: torch.Tensor | None = None,
                 gate_scale: torch.Tensor | None = None, up_scale: torch.Tensor | None = None,
                 out_dtype: torch.dtype | None = None, save: bool = False):
    """act(x w_gate^T) * (x w_up^T) in one kernel: x (..., K), w_gate and w_up
    (F, K); types and scales as ``linear``. Returns h (..., F), with save=True
    (h, g, u), g and u the two projections for gated_linear_backward."""
    op = "gated_linear"
    dev = _device(op, x, w_gate, w_up, x_scale, gate_scale, up_scale)
    px, ldx, T, K = _rows(op, x, "x")
    pg, ldg, F, _ = _rows(op, w_gate, "w_gate", K, None, x.dtype)
    pu, ldu, _, _ = _rows(op, w_up, "w_up", K, F, x.dtype)
    od = _out_type(op, x.dtype, out_dtype, (x_scale, gate_scale, up_scale))
    ty, to = _type(op, x.dtype), _type(op, od)
    h = _new(x, F, od)
    g, u = (_new(x, F, od), _new(x, F, od)) if save else (None, None)
    a = GatedArgs(px, pg, pu, _vec(op, x_scale, "x_scale", T),
                  _vec(op, gate_scale, "gate_scale", F), _vec(op, up_scale, "up_scale", F),
                  h.data_ptr(), None if g is None else g.data_ptr(),
                  None if u is None else u.data_ptr(), ldx, ldg, ldu, F, F, F, T, K, F, ty, to,
                  _act(op, act))
    _run(_gated, _gated_ws, a, dev)
    return (h, g, u) if save else h


def gated_linear_backward(dh: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor,
                          w_up: torch.Tensor, g: torch.Tensor, u: torch.Tensor, *,
                          act: str = "silu", dx: bool = True, dw: bool = True):
    """(dx, dw_gate, dw_up) of gated_linear for fp16 or bf16 matrices; g and u
    (..., F) are what gated_linear(save=True) returned. dx=False or dw=False
    leave gradients out (None)."""
    op = "gated_linear_backward"
    dev = _device(op, dh, x, w_gate, w_up, g, u)
    px, ldx, T, K = _rows(op, x, "x")
    pg, ldg, F, _ = _rows(op, w_gate, "w_gate", K, None, x.dtype)
    pu, ldu, _, _ = _rows(op, w_up, "w_up", K, F, x.dtype)
    if dh.shape[:-1] != x.shape[:-1] or g.shape != dh.shape or u.shape != dh.shape:
        raise _err(op, "dh, g and u must have one shape, with x's rows")
    pd, ldd, _, _ = _rows(op, dh, "dh", F, T, x.dtype)
    pgv, ldgv, _, _ = _rows(op, g, "g", F, T, x.dtype)
    puv, lduv, _, _ = _rows(op, u, "u", F, T, x.dtype)
    gx = _like(x) if dx else None
    gg, gu = (torch.empty((F, K), dtype=x.dtype, device=x.device) for _ in range(2)) if dw \
        else (None, None)
    a = GatedBackwardArgs(pd, pgv, puv, px, pg, pu, None if gx is None else gx.data_ptr(),
                          None if gg is None else gg.data_ptr(),
                          None if gu is None else gu.data_ptr(), ldd, ldgv, lduv, ldx, ldg, ldu,
                          K, K, K, T, K, F, _type(op, x.dtype), _act(op, act))
    _run(_gated_bwd, _gated_bwd_ws, a, dev)
    return gx, gg, gu


def blocks_status(device: torch.device | int | None = None) -> None:
    """Synchronises the device's current stream and raises if a matrix
    product's pipeline gave up waiting since the last call (its result is then
    unspecified)."""
    dev = torch.device("cuda", device) if isinstance(device, int) else device
    with torch.cuda.device(dev):
        _check(_status(torch.cuda.current_stream().cuda_stream))
