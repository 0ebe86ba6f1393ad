"""Feed-forward operators over rows of features (pixels of a grid, tokens of a
sequence), the kernels of libbvml_blocks.so (include/bvml_blocks.h):

  rms_norm, rms_norm_e4m3   s = x + residual, s / sqrt(mean(s^2) + eps) * weight,
                            in the rows' type or in 8 bits with a scale a row
  linear                    act(x w^T + bias) + residual
  gated_linear              act(x w_gate^T) * (x w_up^T)

each with its backward pass as a function of its own (``*_backward``): the
operators take no part in torch's autograd, and refuse inputs that require
gradients while it records, that carry a forward-mode tangent, or that belong to a trace,
a transform (vmap, torch.func) or a tensor class that torch dispatches on.

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

import importlib.machinery
import importlib.util
import os

import torch

from ._capi import LIB_PATH

BLOCKS_LIB_PATH = os.path.join(os.path.dirname(LIB_PATH), "libbvml_blocks.so")


def _load_binding():
    from .build import blocks_torch_path

    path = blocks_torch_path(torch.__version__)
    if not os.path.exists(path):
        raise ImportError(
            f"brovisionml_b200: binding not built for torch {torch.__version__} and this Python "
            f"({path} missing); run `python brovisionml_b200/build.py` (nvcc for sm_100a)")
    loader = importlib.machinery.ExtensionFileLoader("_blocks_torch", path)
    spec = importlib.util.spec_from_loader("_blocks_torch", loader)
    module = importlib.util.module_from_spec(spec)
    loader.exec_module(module)
    return module


class _Unloaded:
    """Stands for the binding until the first call of an operator here, which loads it: it
    is bound to one torch and one Python, and without it the rest of the package works."""

    def __getattr__(self, name):
        global _binding
        if name.startswith("__"):  # somebody looking around, not a call
            raise AttributeError(name)
        _binding = _load_binding()
        return getattr(_binding, name)


_binding = _Unloaded()

BLOCK_ACTIVATIONS = {"none": 0, "relu": 1, "sigmoid": 2, "tanh": 3, "silu": 4, "gelu": 5}


def _act(op: str, act: str) -> int:
    code = BLOCK_ACTIVATIONS.get(act)
    if code is None:
        raise RuntimeError(f"dsine ops: {op}: unknown activation {act!r}")
    return code


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
             eps: float = 1e-6):
    """y = s / sqrt(mean(s^2) + eps) * weight with s = x + residual, row by row.
    x and residual (..., K) fp32, fp16 or bf16; weight (K) of that type or
    fp32. Returns y, or with a residual (y, s), both of x's type; the norm
    is taken of the unrounded sum."""
    return _binding.rms_norm(x, weight, residual, eps)


def rms_norm_e4m3(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
                  *, eps: float = 1e-6):
    """rms_norm with y in 8 bits, as ``linear`` and ``gated_linear`` take it:
    (q, scale) or, with a residual, (q, scale, s); q (..., K) float8_e4m3fn, scale (...)
    fp32, y ~ q * scale[..., None]. The row's largest magnitude becomes 448
    (zeros and scale 1 where that magnitude is below 2^-110; a row with NaN or infinities has
    a NaN scale)."""
    return _binding.rms_norm_e4m3(x, weight, residual, eps)


def rms_norm_backward(dy: torch.Tensor, s: torch.Tensor, weight: torch.Tensor,
                      dsum: torch.Tensor | None = None, *, eps: float = 1e-6):
    """(dx, dweight) of rms_norm: s is the sum its forward pass returned (x
    without a residual), dsum the gradient of that sum where it went on as
    the residual stream. dx is the gradient of x and of the residual alike."""
    return _binding.rms_norm_backward(dy, s, weight, dsum, eps)


def pack_weight_e4m3(weight: torch.Tensor):
    """(N, K) weights -> (q, scale) for ``linear`` / ``gated_linear``: e4m3 values
    and one fp32 scale an output feature, weight ~ q * scale[:, None]."""
    w = weight.detach().float()
    scale = w.abs().amax(1) / 448.0
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return (w / scale[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
           act: str = "none", residual: torch.Tensor | None = None,
           x_scale: torch.Tensor | None = None, w_scale: torch.Tensor | None = None,
           out_dtype: torch.dtype | None = None, save: bool = False):
    """act(x weight^T + bias) + residual on the tensor cores, fp32 accumulation,
    one rounding. x (..., K), weight (N, K), bias (N) fp32, residual (..., N) of
    the output's type: the inputs' type or fp32 (``out_dtype``). e4m3 inputs come
    with x_scale (...) and w_scale (N), and give bf16 unless out_dtype says
    otherwise. act: none, relu, sigmoid, tanh, silu, gelu (x Phi(x)). Returns
    y (..., N), with save=True (y, z), z the pre-activation for linear_backward."""
    return _binding.linear(x, weight, bias, _act("linear", act), residual, x_scale, w_scale,
                           out_dtype, save)


def linear_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                    z: torch.Tensor | None = None, *, act: str = "none", bias: bool = False,
                    dx: bool = True, dw: bool = True):
    """(dx, dweight, dbias) of linear for fp16 or bf16 matrices: dy (..., N), x
    (..., K), weight (N, K), z (..., N) the pre-activation that linear(save=True)
    returned (None without an activation). dbias is fp32, None unless ``bias``; dx=False
    or dw=False leave that gradient out (None). The residual's gradient is dy."""
    return _binding.linear_backward(dy, x, weight, z, _act("linear_backward", act), bias, dx, dw)


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, *,
                 act: str = "silu", x_scale: torch.Tensor | None = None,
                 gate_scale: torch.Tensor | None = None, up_scale: torch.Tensor | None = None,
                 out_dtype: torch.dtype | None = None, save: bool = False):
    """act(x w_gate^T) * (x w_up^T) in one kernel: x (..., K), w_gate and w_up
    (F, K); types and scales as ``linear``. Returns h (..., F), with save=True
    (h, g, u), g and u the two projections for gated_linear_backward."""
    return _binding.gated_linear(x, w_gate, w_up, _act("gated_linear", act), x_scale, gate_scale,
                                 up_scale, out_dtype, save)


def gated_linear_backward(dh: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor,
                          w_up: torch.Tensor, g: torch.Tensor, u: torch.Tensor, *,
                          act: str = "silu", dx: bool = True, dw: bool = True):
    """(dx, dw_gate, dw_up) of gated_linear for fp16 or bf16 matrices; g and u
    (..., F) are what gated_linear(save=True) returned. dx=False or dw=False
    leave gradients out (None)."""
    return _binding.gated_linear_backward(dh, x, w_gate, w_up, g, u,
                                          _act("gated_linear_backward", act), dx, dw)


def blocks_status(device: torch.device | int | None = None) -> None:
    """Synchronises the device's current stream and raises if a matrix
    product's pipeline gave up waiting since the last call (its result is then
    unspecified)."""
    from . import _blocks_capi

    dev = torch.device("cuda", device) if isinstance(device, int) else device
    with torch.cuda.device(dev):
        _blocks_capi.check(_blocks_capi.status(torch.cuda.current_stream().cuda_stream))
