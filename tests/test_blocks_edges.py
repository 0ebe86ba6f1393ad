"""CPU tests of the feed-forward operators at the edges of what their documents allow."""
import ctypes
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig

import pytest
import torch
import torch.autograd.forward_ad as fwad

import brovisionml_b200 as bv
from brovisionml_b200 import _blocks_capi as B
from test_blocks_api import (BF16, E4M3, EINVAL, EWORKSPACE, at, err, gated_args, linear_args)


@pytest.mark.parametrize("x,x_scale", [(None, None), (at(0), at(5))])
def test_empty_batches_in_8_bits(x, x_scale):
    """T = 0 rows are fine in 8 bits too, their (empty) scales null or not; the weights'
    scales are needed all the same."""
    a = linear_args(T=0, x=x, y=None, in_type=E4M3, x_scale=x_scale, w_scale=at(6))
    assert B.blocks_lib.bvml_linear(ctypes.byref(a), None, 0, None) == 0, err()
    assert B.blocks_lib.bvml_linear_workspace_bytes(ctypes.byref(a)) == 0
    a = gated_args(T=0, x=x, h=None, in_type=E4M3, out_type=BF16, x_scale=x_scale,
                   gate_scale=at(6), up_scale=at(7))
    assert B.blocks_lib.bvml_gated_linear(ctypes.byref(a), None, 0, None) == 0, err()
    a = linear_args(T=0, x=x, y=None, in_type=E4M3, x_scale=x_scale)
    assert B.blocks_lib.bvml_linear(ctypes.byref(a), None, 0, None) == EINVAL
    assert "need their scales" in err()
    a = linear_args(T=1, in_type=E4M3, w_scale=at(6))
    assert B.blocks_lib.bvml_linear(ctypes.byref(a), None, 0, None) == EINVAL
    assert "need their scales" in err()


def calls(t, w, v):
    """Every operator, with t among its tensors (rows for the inner axis of 8)."""
    return [lambda: bv.rms_norm(t, v), lambda: bv.rms_norm(w, v, t),
            lambda: bv.rms_norm_e4m3(t, v), lambda: bv.rms_norm_backward(w, t, v),
            lambda: bv.rms_norm_backward(t, w, v), lambda: bv.linear(t, w),
            lambda: bv.linear(w, t), lambda: bv.linear(w, w, residual=t[:, :6]),
            lambda: bv.linear_backward(t[:, :6], w, w), lambda: bv.gated_linear(w, w, t),
            lambda: bv.gated_linear_backward(w[:, :6], w, w, w, w[:, :6], t[:, :6])]


def test_what_torch_follows_is_refused():
    """Forward-mode tangents, traces, transforms and tensor classes would be dropped without
    a word: refused, whichever argument carries them."""
    w, v = torch.ones(6, 8), torch.ones(8)
    with fwad.dual_level():
        t = fwad.make_dual(torch.ones(6, 8), torch.ones(6, 8))
        for call in calls(t, w, v):
            with pytest.raises(RuntimeError, match="dsine ops: .*forward-mode"):
                call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            bv.linear(t, w)  # no_grad() does not end forward mode
        with torch.inference_mode(), pytest.raises(RuntimeError, match="CUDA-resident"):
            bv.linear(t, w)  # ... which inference_mode() does
        with pytest.raises(RuntimeError, match="CUDA-resident"):
            bv.linear(fwad.unpack_dual(t).primal, w)

    def inside(t):
        for call in calls(t, w, v):
            with pytest.raises(RuntimeError, match="dsine ops: .*(transforms|autograd|forward)"):
                call()
        return t.sum()

    torch.vmap(inside)(torch.ones(2, 6, 8))
    torch.func.grad(inside)(torch.ones(6, 8))
    torch.func.jvp(inside, (torch.ones(6, 8),), (torch.ones(6, 8),))
    torch.func.functionalize(inside)(torch.ones(6, 8))

    class Named(torch.Tensor):
        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with pytest.raises(RuntimeError, match="plain tensors"):
        bv.linear(torch.Tensor._make_subclass(Named, torch.ones(6, 8)), w)

    def traced(t):
        with pytest.raises(RuntimeError, match="dsine ops: linear: cannot be traced"):
            bv.linear(w, w)
        return t + 1

    torch.jit.trace(traced, torch.ones(2), check_trace=False)
    from torch.fx.experimental.proxy_tensor import make_fx
    make_fx(traced)(torch.ones(2))
    with pytest.raises(RuntimeError, match="CUDA-resident"):  # and after all that as before
        bv.linear(w, w)


def test_lazy_values_are_refused():
    """Tensors whose memory does not hold their values: a negation that torch has put off
    (the imaginary part of a conjugate), zeros without memory."""
    w, v = torch.ones(6, 8), torch.ones(8)
    for t in (torch._neg_view(torch.ones(6, 8)), torch._efficientzerotensor(6, 8)):
        for call in calls(t, w, v):
            with pytest.raises(RuntimeError, match="dsine ops: .*hold its values"):
                call()
    with pytest.raises(RuntimeError, match="CUDA-resident"):
        bv.linear(torch._neg_view(torch.ones(6, 8)).resolve_neg(), w)


class Untrue:
    def __bool__(self):
        raise ValueError("neither true nor false")


def test_flags_without_a_truth_value_raise_their_error():
    """... and not a SystemError from a result returned beside a pending exception."""
    w = torch.ones(6, 8)
    d = w[:, :6]
    for call in (lambda f: bv.linear(w, w, save=f), lambda f: bv.gated_linear(w, w, w, save=f),
                 lambda f: bv.linear_backward(d, w, w, bias=f),
                 lambda f: bv.linear_backward(d, w, w, dx=f),
                 lambda f: bv.linear_backward(d, w, w, dw=f),
                 lambda f: bv.gated_linear_backward(d, w, w, w, d, d, dx=f),
                 lambda f: bv.gated_linear_backward(d, w, w, w, d, d, dw=f)):
        with pytest.raises(ValueError, match="neither true nor false"):
            call(Untrue())
        with pytest.raises(RuntimeError, match="ambiguous"):
            call(torch.ones(2))
        with pytest.raises(RuntimeError, match="CUDA-resident"):
            call(True)


def test_the_package_works_without_these_operators(tmp_path):
    """A missing library or binding of the feed-forward operators is an ImportError of their
    first call, and takes nothing else of the package with it."""
    src = os.path.dirname(os.path.abspath(bv.__file__))
    dst = tmp_path / "brovisionml_b200"
    (dst / "_lib").mkdir(parents=True)
    for f in os.listdir(src):
        if f.endswith(".py"):
            shutil.copy(os.path.join(src, f), dst / f)
    os.symlink(os.path.join(src, "_lib", "libbvml_dsine.so"), dst / "_lib" / "libbvml_dsine.so")
    code = """
import brovisionml_b200 as bv, torch
assert bv.abi_version() > 0 and bv.refine_workspace_bytes(1, 8, 8) > 0 and callable(bv.refine)
w = torch.ones(6, 8)
q, s = bv.pack_weight_e4m3(w)
for call in (lambda: bv.linear(w, w), lambda: bv.rms_norm(w, w[0]), lambda: bv.blocks_status(None)):
    for _ in range(2):
        try:
            call()
        except ImportError as e:
            assert 'not built' in str(e), e
        else:
            raise SystemExit('no ImportError')
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=tmp_path, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_the_binding_belongs_to_one_torch_and_python(monkeypatch):
    """Its file name has both versions: the build makes one for each, and another version's
    is never loaded."""
    from brovisionml_b200 import blocks, build

    assert build.torch_version() == torch.__version__
    path = build.blocks_torch_path(torch.__version__)
    assert os.path.exists(path)
    assert sysconfig.get_config_var("SOABI") in path and torch.__version__ in path
    assert blocks._load_binding().__file__ == path
    monkeypatch.setattr(torch, "__version__", "0.1.2")
    with pytest.raises(ImportError, match="not built for torch 0.1.2"):
        blocks._load_binding()
    monkeypatch.undo()
    monkeypatch.setattr(sysconfig, "get_config_var", lambda name: "cpython-27-x")
    with pytest.raises(ImportError, match="not built for torch"):
        blocks._load_binding()


@pytest.fixture
def fake_build(tmp_path, monkeypatch):
    """The build script with its outputs under tmp_path and its commands recorded, not run;
    fake_build.fails: a text whose commands fail."""
    spec = importlib.util.spec_from_file_location("fake_build", os.path.join(
        os.path.dirname(os.path.abspath(bv.__file__)), "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    for name in [n for n in vars(build) if n.isupper()]:
        v = getattr(build, name)
        if isinstance(v, str) and name not in ("HERE", "ROOT", "CSRC", "BLOCKS"):
            monkeypatch.setattr(build, name, str(tmp_path / os.path.relpath(v, build.HERE)))
    build.done, build.fails = [], "nothing"

    def run(cmd, **kw):
        build.done.append(cmd)
        bad = any(build.fails in a for a in cmd)
        if not bad:
            open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, int(bad), "", "no")

    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "_nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    return build


def test_build_without_torch(fake_build, monkeypatch, capsys):
    """The C and C++ libraries need no torch: the binding alone is left out."""
    monkeypatch.setattr(fake_build.importlib.util, "find_spec", lambda name: None)
    fake_build.build()
    for lib in (fake_build.LIB, fake_build.CHECKED_LIB, fake_build.BRIDGE, fake_build.BLOCKS_LIB,
                fake_build.BLOCKS_CHECKED_LIB):
        assert os.path.exists(lib)
    assert "binding is left out" in capsys.readouterr().err
    assert not any("blocks_torch" in a for cmd in fake_build.done for a in cmd)


@pytest.mark.parametrize("fails", ["blocks_torch.cpp", "gemm_tile_nt.cu"])
def test_build_makes_the_refinement_first(fake_build, fails):
    """What fails in the feed-forward operators' part is an error, after the refinement's
    libraries are there."""
    fake_build.fails = fails
    with pytest.raises(RuntimeError, match=fails):
        fake_build.build()
    assert all(os.path.exists(p) for p in (fake_build.LIB, fake_build.CHECKED_LIB,
                                           fake_build.BRIDGE))
    fake_build.fails, fake_build.done = "nothing", []
    fake_build.build()
    assert os.path.exists(fake_build.BLOCKS_LIB)
    assert os.path.exists(fake_build.blocks_torch_path(torch.__version__))
    fake_build.done = []
    fake_build.build()
    assert not fake_build.done  # all of it is up to date


def test_neighbouring_columns_of_one_buffer_are_accepted():
    """An output in the columns beside its input (64 + 32 elements of rows of 96), its last
    byte before the next row and its first after the input's last: past the overlap checks
    and turned down only for want of a workspace, before any launch. One element nearer to
    either side is an overlap."""
    lib = B.blocks_lib
    # an input on an odd address is laid out anew in the workspace
    base = at(0) + 2

    def call(off, ldx=96):
        a = linear_args(x=base, ldx=ldx, ldy=ldx, y=base + off)
        return (lib.bvml_linear(ctypes.byref(a), None, 0, None),
                lib.bvml_linear_workspace_bytes(ctypes.byref(a)))

    rc, need = call(128)
    assert rc == EWORKSPACE and need > 0, err()
    for off, ldx in ((126, 96), (130, 96), (128, 95), (-62, 96), (-66, 96)):
        rc, need = call(off, ldx)
        assert rc == EINVAL and need == 0 and "y overlaps x" in err(), (off, ldx)
    rc, need = call(-64)  # before it, in the columns of the row before
    assert rc == EWORKSPACE and need > 0, err()


@pytest.mark.parametrize("vector", ["bias", "w_scale", "gate_scale", "up_scale"])
def test_vectors_off_16_bytes_go_through_the_workspace(vector):
    """A bias or scales that start on no 16 bytes are laid out anew like rows that do not (in
    place they would be read one element after the other); few rows read them as they are."""
    lib = B.blocks_lib
    if vector in ("gate_scale", "up_scale"):
        make, name = gated_args, "bvml_gated_linear"
        kw = dict(in_type=E4M3, x_scale=at(6), gate_scale=at(7), up_scale=at(8))
    else:
        make, name = linear_args, "bvml_linear"
        kw = dict(in_type=E4M3, x_scale=at(6), w_scale=at(7), bias=at(8))
    size, fn = getattr(lib, name + "_workspace_bytes"), getattr(lib, name)
    assert size(ctypes.byref(make(T=300, **kw))) == 0
    kw[vector] += 4
    a = make(T=300, **kw)
    assert size(ctypes.byref(a)) == 256  # 32 floats
    assert fn(ctypes.byref(a), None, 0, None) == EWORKSPACE
    assert size(ctypes.byref(make(T=7, **kw))) == 0
