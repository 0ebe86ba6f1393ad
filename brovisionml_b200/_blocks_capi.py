"""ctypes binding of libbvml_blocks.so (the C ABI in include/bvml_blocks.h), for
callers with device pointers of their own. ``blocks.py`` has the operators on
torch tensors.

The library must have been built in-tree (``python brovisionml_b200/build.py``);
a missing library is an ImportError, never a silent fallback.
"""
from __future__ import annotations

import ctypes
import os

from ._capi import BVML_OK
from .blocks import BLOCKS_LIB_PATH

BVML_BF16 = 2
BVML_E4M3 = 3
BVML_EWORKSPACE = 4

# Every symbol include/bvml_blocks.h declares (checked by the CPU test suite).
EXPORTS = ("bvml_blocks_last_error", "bvml_blocks_version", "bvml_blocks_status",
           "bvml_blocks_wait_limit",
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


last_error = _bind("bvml_blocks_last_error", ctypes.c_char_p, [])
_bind("bvml_blocks_version", _i, [])
status = _bind("bvml_blocks_status", _i, [_vp])
_bind("bvml_blocks_wait_limit", ctypes.c_uint, [ctypes.c_uint])
_bind("bvml_rms_norm", _i, [_vp, _ll, _vp, _ll, _vp, _i, _i, _i, _i, _f, _vp, _ll, _vp,
                                    _ll, _vp])
_bind("bvml_rms_norm_e4m3", _i, [_vp, _ll, _vp, _ll, _vp, _i, _i, _i, _i, _f, _vp,
                                              _ll, _vp, _vp, _ll, _vp])
_bind("bvml_rms_norm_backward_workspace_bytes", _sz, [_i, _i])
_bind("bvml_rms_norm_backward", _i, [_vp, _ll, _vp, _ll, _vp, _vp, _ll, _i, _i, _i,
                                                 _i, _f, _vp, _ll, _vp, _vp, _sz, _vp])


def _bind_args(name, struct):
    """An entry point that takes a structure, and its workspace's size."""
    p = ctypes.POINTER(struct)
    _bind(name, _i, [p, _vp, _sz, _vp])
    _bind(name + "_workspace_bytes", _sz, [p])


_bind_args("bvml_linear", LinearArgs)
_bind_args("bvml_linear_backward", LinearBackwardArgs)
_bind_args("bvml_gated_linear", GatedArgs)
_bind_args("bvml_gated_linear_backward", GatedBackwardArgs)


def check(rc: int) -> None:
    if rc != BVML_OK:
        msg = last_error().decode("utf-8", "replace")
        raise RuntimeError(msg or f"dsine ops: failed with status {rc}")
