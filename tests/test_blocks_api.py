"""CPU tests of the feed-forward operators' C ABI and Python entry points: every
declared symbol is exported, and bad arguments are refused with the
library's error wording before any CUDA call."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import brovisionml_b200 as bv
from brovisionml_b200 import _blocks_capi as B

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "bvml_blocks.h")
EINVAL, EWORKSPACE = 1, 4
F32, F16, BF16, E4M3 = 0, 1, 2, 3


def at(n):
    """A fake device address: never dereferenced, 64 MiB apart."""
    return 0x100000000 + n * (64 << 20)


def err():
    return B.blocks_lib.bvml_blocks_last_error().decode()


def test_header_symbols_exported():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    syms = sorted(set(re.findall(r"\b(bvml_[a-z0-9_]+)\s*\(", text)))
    assert sorted(B.EXPORTS) == syms
    out = subprocess.run(["nm", "-D", "--defined-only", bv.BLOCKS_LIB_PATH], capture_output=True,
                         text=True, check=True).stdout
    assert set(re.findall(r" T (bvml_\w+)", out)) == set(syms)
    assert B.blocks_lib.bvml_blocks_version() == 1


def test_struct_sizes_match_the_header(tmp_path):
    """ctypes' structures have the compiler's layout."""
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "bvml_blocks.h"\nint main(void) { printf("%zu '
                   '%zu %zu %zu", sizeof(bvml_linear_args), sizeof(bvml_linear_backward_args), '
                   'sizeof(bvml_gated_args), sizeof(bvml_gated_backward_args)); }\n')
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)],
                   check=True)
    sizes = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    assert [int(v) for v in sizes] == [ctypes.sizeof(s) for s in (
        B.LinearArgs, B.LinearBackwardArgs, B.GatedArgs, B.GatedBackwardArgs)]


def linear_args(**kw):
    a = dict(x=at(0), w=at(1), y=at(2), ldx=64, ldw=64, ldr=32, ldy=32, ldz=32, T=16, K=64, N=32,
             in_type=BF16, out_type=BF16, act=0)
    a.update(kw)
    return B.LinearArgs(**a)


@pytest.mark.parametrize("change,what", [
    (dict(x=None), "x is null"),
    (dict(w=None), "w is null"),
    (dict(y=None), "y is null"),
    (dict(x=at(0) + 1), "x is not aligned"),
    (dict(ldx=63), "x has a row stride below"),
    (dict(ldy=31), "y has a row stride below"),
    (dict(T=-1), "bad shape"),
    (dict(K=0), "bad shape"),
    (dict(N=0), "bad shape"),
    (dict(in_type=F32), "inputs must be"),
    (dict(out_type=F16), "output must be"),
    (dict(out_type=E4M3), "output must be"),
    (dict(act=6), "unknown activation"),
    (dict(act=-1), "unknown activation"),
    (dict(in_type=E4M3), "need their scales"),
    (dict(x_scale=at(5)), "scales belong to"),
    (dict(y=at(0) + 128), "y overlaps x"),
    (dict(y=at(1)), "y overlaps w"),
    (dict(residual=at(2)), "y overlaps residual"),
    (dict(bias=at(2) + 4), "y overlaps bias"),
    (dict(z=at(2)), "z overlaps y"),
])
def test_linear_refusals(change, what):
    rc = B.blocks_lib.bvml_linear(ctypes.byref(linear_args(**change)), None, 0, None)
    assert rc == EINVAL and err().startswith("dsine ops: linear: ") and what in err(), err()
    assert B.blocks_lib.bvml_linear_workspace_bytes(ctypes.byref(linear_args(**change))) == 0


def test_columns_of_one_buffer_do_not_overlap():
    """Output beside its input in one wider buffer: refused only where they meet
    (the call that gets past the checks asks for no more than a workspace)."""
    def over(ldx, off):
        a = linear_args(ldx=ldx, ldy=ldx, y=at(0) + off)
        rc = B.blocks_lib.bvml_linear(ctypes.byref(a), None, 0, None)
        return rc == EINVAL and "overlaps" in err()

    assert over(95, 128)         # 64 + 32 columns in rows of 95
    assert over(96, 126)         # starts inside x
    # odd K, whose rows start on no 16-byte boundary, needs a workspace: turned
    # down there, after the overlap checks and before any launch
    b = linear_args(K=63, ldx=95, ldw=63, ldy=95, y=at(0) + 126)
    if B.blocks_lib.bvml_linear_workspace_bytes(ctypes.byref(b)):
        assert B.blocks_lib.bvml_linear(ctypes.byref(b), None, 0, None) == EWORKSPACE


def gated_args(**kw):
    a = dict(x=at(0), w_gate=at(1), w_up=at(2), h=at(3), ldx=64, ldw_gate=64, ldw_up=64, ldh=32,
             ldg=32, ldu=32, T=16, K=64, F=32, in_type=F16, out_type=F16, act=4)
    a.update(kw)
    return B.GatedArgs(**a)


@pytest.mark.parametrize("change,what", [
    (dict(act=0), "unknown activation"),
    (dict(g=at(4)), "kept together"),
    (dict(w_up=None), "w_up is null"),
    (dict(ldw_up=60), "w_up has a row stride below"),
    (dict(F=0), "bad shape"),
    (dict(in_type=E4M3, x_scale=at(6), gate_scale=at(7)), "need their scales"),
    (dict(up_scale=at(7)), "scales belong to"),
    (dict(h=at(2) + 2), "h overlaps w_up"),
    (dict(g=at(4), u=at(4) + 64), "u overlaps g"),
])
def test_gated_refusals(change, what):
    rc = B.blocks_lib.bvml_gated_linear(ctypes.byref(gated_args(**change)), None, 0, None)
    assert rc == EINVAL and err().startswith("dsine ops: gated_linear: ") and what in err(), err()


def linear_backward_args(**kw):
    a = dict(dy=at(0), z=at(1), x=at(2), w=at(3), dx=at(4), dw=at(5), dbias=at(6), lddy=32, ldz=32,
             ldx=64, ldw=64, lddx=64, lddw=64, T=16, K=64, N=32, type=BF16, act=4)
    a.update(kw)
    return B.LinearBackwardArgs(**a)


@pytest.mark.parametrize("change,what", [
    (dict(z=None), "z is null"),
    (dict(act=0), "z belongs to an activation"),
    (dict(type=F32), "must be fp16 or bf16"),
    (dict(type=E4M3), "must be fp16 or bf16"),
    (dict(dx=at(5)), "dw overlaps dx"),
    (dict(dx=at(0)), "dx overlaps dy"),
    (dict(dbias=at(6) + 2), "dbias is not aligned"),
    (dict(lddw=63), "dw has a row stride below"),
])
def test_linear_backward_refusals(change, what):
    a = linear_backward_args(**change)
    rc = B.blocks_lib.bvml_linear_backward(ctypes.byref(a), at(8), 1 << 30, None)
    assert rc == EINVAL and err().startswith("dsine ops: linear_backward: ") and what in err(), \
        err()


def gated_backward_args(**kw):
    a = dict(dh=at(0), g=at(1), u=at(2), x=at(3), w_gate=at(4), w_up=at(5), dx=at(6), dw_gate=at(7),
             dw_up=at(8), lddh=32, ldg=32, ldu=32, ldx=64, ldw_gate=64, ldw_up=64, lddx=64,
             lddw_gate=64, lddw_up=64, T=16, K=64, F=32, type=F16, act=4)
    a.update(kw)
    return B.GatedBackwardArgs(**a)


@pytest.mark.parametrize("change,what", [
    (dict(act=0), "unknown activation"),
    (dict(dw_up=None), "computed together"),
    (dict(type=F32), "must be fp16 or bf16"),
    (dict(u=None), "u is null"),
    (dict(dw_up=at(7) + 64 * 2), "dw_up overlaps dw_gate"),
])
def test_gated_backward_refusals(change, what):
    a = gated_backward_args(**change)
    rc = B.blocks_lib.bvml_gated_linear_backward(ctypes.byref(a), at(9), 1 << 30, None)
    assert rc == EINVAL and what in err(), err()


def test_workspace_refusals():
    """Too small, missing or misaligned workspaces are refused before a launch."""
    lib = B.blocks_lib
    for a, fn, size in (
            (linear_backward_args(), lib.bvml_linear_backward,
             lib.bvml_linear_backward_workspace_bytes),
            (gated_backward_args(), lib.bvml_gated_linear_backward,
             lib.bvml_gated_linear_backward_workspace_bytes)):
        need = size(ctypes.byref(a))
        assert need > 0
        assert fn(ctypes.byref(a), None, 0, None) == EWORKSPACE
        assert fn(ctypes.byref(a), at(10), need - 1, None) == EWORKSPACE and "small" in err()
        assert fn(ctypes.byref(a), at(10) + 128, need, None) == EWORKSPACE and "aligned" in err()
    need = lib.bvml_rms_norm_backward_workspace_bytes(16, 64)
    args = (at(0), 64, at(1), 64, at(2), None, 0, 16, 64, BF16, F32, 1e-6, at(3), 64, at(4))
    assert lib.bvml_rms_norm_backward(*args, at(5), need - 1, None) == EWORKSPACE
    assert lib.bvml_rms_norm_backward(*args, at(5) + 16, need, None) == EWORKSPACE


@pytest.mark.parametrize("change,what", [
    (dict(dtype=E4M3), "rows must be"),
    (dict(wtype=F16), "weights must be"),
    (dict(T=-1), "bad shape"),
    (dict(K=0), "bad shape"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(w=None), "weight is null"),
    (dict(x=None), "x is null"),
    (dict(sum=at(4)), "residual's addition"),
    (dict(r=at(1), sum=at(1)), "sum overlaps residual"),
    (dict(y=at(0) + 64), "y overlaps x"),
    (dict(ldx=63), "x has a row stride below"),
])
def test_norm_refusals(change, what):
    a = dict(x=at(0), r=None, w=at(2), T=16, K=64, dtype=BF16, wtype=F32, eps=1e-6, y=at(3),
             sum=None, ldx=64)
    a.update(change)
    rc = B.blocks_lib.bvml_rms_norm(a["x"], a["ldx"], a["r"], 64, a["w"], a["T"], a["K"],
                                    a["dtype"], a["wtype"], a["eps"], a["y"], 64, a["sum"], 64,
                                    None)
    assert rc == EINVAL and err().startswith("dsine ops: rms_norm: ") and what in err(), err()
    rc = B.blocks_lib.bvml_rms_norm_e4m3(a["x"], a["ldx"], a["r"], 64, a["w"], a["T"], a["K"],
                                         a["dtype"], a["wtype"], a["eps"], a["y"], 64, at(9),
                                         a["sum"], 64, None)
    assert rc == EINVAL and err().startswith("dsine ops: rms_norm_e4m3: ") and what in err(), err()


def test_norm_scale_and_backward_refusals():
    lib = B.blocks_lib
    rc = lib.bvml_rms_norm_e4m3(at(0), 64, None, 0, at(2), 16, 64, BF16, F32, 1e-6, at(3), 64,
                                None, None, 0, None)
    assert rc == EINVAL and "scale is null" in err()
    rc = lib.bvml_rms_norm_e4m3(at(0), 64, None, 0, at(2), 16, 64, BF16, F32, 1e-6, at(3), 64,
                                at(3) + 64, None, 0, None)
    assert rc == EINVAL and "scale overlaps y" in err()
    rc = lib.bvml_rms_norm_backward(at(0), 64, at(1), 64, at(2), None, 0, 16, 64, BF16, F32, 1e-6,
                                    at(1), 64, at(4), at(5), 1 << 30, None)
    assert rc == EINVAL and "dx overlaps s" in err()


def test_sizes_past_the_indexes_are_refused():
    """Shapes beyond 32-bit indexes or counts of tiles: refused, and no workspace is named."""
    lib, most = B.blocks_lib, (1 << 30) - 64
    for kw in (dict(T=most + 1), dict(K=most + 1), dict(N=2**31 - 1), dict(T=1 << 25, N=1 << 25)):
        kw = dict(ldx=1 << 31, ldw=1 << 31, ldy=1 << 31, ldz=1 << 31) | kw
        a = linear_args(**kw)
        assert lib.bvml_linear(ctypes.byref(a), None, 0, None) == EINVAL and "bad shape" in err()
        assert lib.bvml_linear_workspace_bytes(ctypes.byref(a)) == 0
        a = linear_backward_args(**kw)
        assert lib.bvml_linear_backward(ctypes.byref(a), None, 0, None) == EINVAL
        assert "bad shape" in err()
        assert lib.bvml_linear_backward_workspace_bytes(ctypes.byref(a)) == 0
        kw = {("F" if k == "N" else k): v for k, v in kw.items() if k[:2] != "ld"}
        a = gated_args(**kw)
        assert lib.bvml_gated_linear(ctypes.byref(a), None, 0, None) == EINVAL
        assert "bad shape" in err()
        a = gated_backward_args(**kw)
        assert lib.bvml_gated_linear_backward(ctypes.byref(a), None, 0, None) == EINVAL
        assert "bad shape" in err()
    for T, K in ((most + 1, 64), (16, 2**31 - 1)):
        assert lib.bvml_rms_norm(at(0), 1 << 31, None, 0, at(1), T, K, BF16, F32, 1e-6, at(2),
                                 1 << 31, None, 0, None) == EINVAL and "bad shape" in err()
        assert lib.bvml_rms_norm_backward_workspace_bytes(T, K) == 0


def test_python_refusals():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    with pytest.raises(RuntimeError, match="dsine ops: linear: .*CUDA-resident"):
        bv.linear(x, w)
    with pytest.raises(RuntimeError, match="dsine ops: gated_linear: .*CUDA-resident"):
        bv.gated_linear(x, w, w)
    with pytest.raises(RuntimeError, match="dsine ops: rms_norm: .*CUDA-resident"):
        bv.rms_norm(x, torch.ones(8))
    with pytest.raises(RuntimeError, match="no autograd"):
        bv.linear(x.requires_grad_(), w)
    with pytest.raises(RuntimeError, match="share a device"):
        bv.linear(torch.zeros(4, 8), torch.zeros(6, 8, device="meta"))


def test_pack_weight_e4m3():
    g = torch.Generator().manual_seed(0)
    w = torch.randn(5, 40, generator=g)
    w[3] = 0
    q, scale = bv.pack_weight_e4m3(w)
    assert q.dtype == torch.float8_e4m3fn and scale.dtype == torch.float32
    assert scale[3] == 1 and (q[3].float() == 0).all()
    d = (q.float() * scale[:, None] - w).abs()
    # half a step of e4m3, or of its smallest (2^-9), and the division's rounding
    assert (d <= w.abs() * 2.0 ** -4 * (1 + 1e-6) + scale[:, None] * 2.0 ** -10).all()
