"""The feed-forward operators against plain formulas in 64 bits.

Tolerances, element by element. With u the half step of the output's type
(torch.finfo(t).eps / 2) and e = 2^-24:
 * a sum of n products in 32 bits is off by at most n 2e sum|a b| (2e and not e:
   the tensor cores may cut instead of round);
 * an activation's slope is at most 1.13 (gelu), its evaluation a few e of its
   argument and value;
 * a backward pass rounds dz (dg, du) to 16 bits: u sum|dz w| more;
 * the result is rounded once: u |ref|, or the smallest subnormal's half.
"""
import ctypes
import math

import pytest
import torch

import brovisionml_b200 as bv
from brovisionml_b200 import _blocks_capi as B

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
F16, BF16, F32, E4M3 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn
ACTS = {
    "none": (lambda z: z, lambda z: torch.ones_like(z)),
    "relu": (lambda z: torch.where(z < 0, torch.zeros_like(z), z),
             lambda z: (z > 0).to(z.dtype)),
    "sigmoid": (torch.sigmoid, lambda z: torch.sigmoid(z) * torch.sigmoid(-z)),
    "tanh": (torch.tanh, lambda z: 1 - torch.tanh(z) ** 2),
    "silu": (lambda z: z * torch.sigmoid(z),
             lambda z: torch.sigmoid(z) * (1 + z * torch.sigmoid(-z))),
    "gelu": (lambda z: 0.5 * z * (1 + torch.erf(z / math.sqrt(2))),
             lambda z: 0.5 * (1 + torch.erf(z / math.sqrt(2)))
             + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)),
}


def half(dt):
    return torch.finfo(dt).eps / 2


def rnd(*shape, dt=F32, scale=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * len(shape) + sum(shape))
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dt)


def close(got, ref, tol, name=""):
    """|got - ref| within tol and the output's rounding, everywhere."""
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    lim = tol + half(got.dtype) * (ref.abs() + tol) + torch.finfo(got.dtype).tiny * half(got.dtype) * 2
    bad = ~((got.double() - ref).abs() <= lim)
    assert not bad.any(), (name, int(bad.sum()), got.double()[bad][:4], ref[bad][:4])


def product(x, w, xs=None, ws=None):
    """x w^T in 64 bits, and the bound of a 32-bit sum's error."""
    a, b = x.double(), w.double()
    if xs is not None:
        a, b = a * xs.double()[..., None], b * ws.double()[:, None]
    n = x.shape[-1] + 4
    return a @ b.T, n * 2 * E * (a.abs() @ b.abs().T)


# ----------------------------------------------------------------------- norm

NORM_SHAPES = [(1, 1), (3, 7), (1, 64), (5, 72), (33, 128), (7, 200), (64, 256), (9, 257),
               (12, 512), (5, 1000), (17, 1024), (3, 1032), (2, 2048), (4, 3001), (6, 4096),
               (3, 4104), (2, 8192), (2, 12000), (3, 16384), (2, 16392), (1, 20001)]


def norm_ref(x, w, r, eps):
    s = x.double() + (r.double() if r is not None else 0)
    rstd = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
    return s, s * rstd * w.double(), rstd


@pytest.mark.parametrize("T,K", NORM_SHAPES)
@pytest.mark.parametrize("dt,wt", [(BF16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("res", [False, True])
def test_rms_norm(T, K, dt, wt, res):
    x, w = rnd(T, K, dt=dt, scale=3), rnd(K, dt=wt, seed=1) + 1
    r = rnd(T, K, dt=dt, seed=2) if res else None
    out = bv.rms_norm(x, w, r, eps=1e-5)
    s, y, _ = norm_ref(x, w, r, 1e-5)
    got = out[0] if res else out
    close(got, y, (K / 2 + 8) * E * y.abs())
    if res:
        assert torch.equal(out[1], (x.float() + r.float()).to(dt))
    again = bv.rms_norm(x, w, r, eps=1e-5)
    assert torch.equal(got, again[0] if res else again)


@pytest.mark.parametrize("T,K", NORM_SHAPES)
@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("res", [False, True])
def test_rms_norm_e4m3(T, K, dt, res):
    x, w = rnd(T, K, dt=dt, scale=3), rnd(K, dt=F32, seed=1) + 1
    r = rnd(T, K, dt=dt, seed=2) if res else None
    q, scale, *s = bv.rms_norm_e4m3(x, w, r, eps=1e-5)
    s64, y, _ = norm_ref(x, w, r, 1e-5)
    top = y.abs().amax(-1)
    assert q.dtype == E4M3 and scale.shape == (T,)
    close(scale, top / 448, (K / 2 + 16) * E * top / 448)
    v = q.double() * scale.double()[:, None]
    lim = (2.0 ** -4 + (K + 32) * E) * y.abs() + scale.double()[:, None] * 2.0 ** -10
    assert ((v - y).abs() <= lim).all()
    assert (q.float().abs().amax(-1) == 448).all()
    if res:
        assert torch.equal(s[0], (x.float() + r.float()).to(dt))


@pytest.mark.parametrize("T,K", NORM_SHAPES + [(700, 64), (1300, 520), (650, 2048)])
@pytest.mark.parametrize("dt,wt", [(BF16, F32), (F16, F16), (F32, F32)])
@pytest.mark.parametrize("res", [False, True])
def test_rms_norm_backward(T, K, dt, wt, res):
    s, w, dy = rnd(T, K, dt=dt, scale=2), rnd(K, dt=wt, seed=1) + 1, rnd(T, K, dt=dt, seed=2)
    ds = rnd(T, K, dt=dt, seed=3) if res else None
    dx, dw = bv.rms_norm_backward(dy, s, w, ds, eps=1e-5)
    _, _, rstd = norm_ref(s, w, None, 1e-5)
    n, dyw = s.double() * rstd, dy.double() * w.double()
    dot = (dyw * n).mean(-1, keepdim=True)
    ref = rstd * (dyw - n * dot) + (ds.double() if res else 0)
    size = rstd * (dyw.abs() + n.abs() * (dyw * n).abs().mean(-1, keepdim=True)) \
        + (ds.double().abs() if res else 0)
    close(dx, ref, (2 * K + 16) * E * size, "dx")
    close(dw, (dy.double() * n).sum(0), (T + K + 16) * E * (dy.double() * n).abs().sum(0), "dw")
    dx2, dw2 = bv.rms_norm_backward(dy, s, w, ds, eps=1e-5)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


def test_rms_norm_backward_against_differences():
    T, K = 6, 40
    x, w, dy = rnd(T, K), rnd(K, seed=1) + 1, rnd(T, K, seed=2)
    dx, dw = bv.rms_norm_backward(dy, x, w, eps=1e-3)
    vx, vw, h = rnd(T, K, seed=5).double(), rnd(K, seed=6).double(), 1e-5

    def loss(sign):
        y = norm_ref(x.double() + sign * h * vx, w.double() + sign * h * vw, None, 1e-3)[1]
        return (dy.double() * y).sum()

    want = (loss(1) - loss(-1)) / (2 * h)
    got = (dx.double() * vx).sum() + (dw.double() * vw).sum()
    assert abs(got - want) <= 1e-5 * (1 + abs(want)) * T * K


def test_rms_norm_special_rows():
    K = 64
    x = rnd(7, K, dt=BF16)
    x[0] = 0
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    x[3] = torch.finfo(BF16).max
    x[4] = 1e-38
    w = torch.ones(K, device="cuda")
    y = bv.rms_norm(x, w)
    assert (y[0] == 0).all() and y[1].isnan().all()
    assert y[2, 5].isnan() and (y[2, :5] == 0).all()  # 1 / inf = 0, inf * 0 = NaN
    assert (y[3] == 0).all()  # the sum of squares is infinite, as in 32 bits
    q, scale = bv.rms_norm_e4m3(x, w)
    assert scale[0] == 1 and (q[0].float() == 0).all()
    assert scale[1].isnan() and q[1].float().isnan().all()
    assert scale[2].isnan() and q[2].float().isnan().all()
    assert scale[4] == 1 and (q[4].float() == 0).all()  # below 2^-110 counts as zero
    z = bv.rms_norm(torch.zeros(2, K, device="cuda"), w, eps=0.0)
    assert z.isnan().all()  # 0 / 0, as the formula has it
    good = bv.rms_norm(x[5:], w)
    assert torch.equal(good, y[5:])


def test_rms_norm_strides_and_shapes():
    big = rnd(20, 3, 300, dt=F16)
    x, r = big[:, 0, 4:204], big[:, 1, 1:201]  # rows 1800 bytes apart; r starts on no 16 bytes
    w = rnd(200, dt=F16)
    y, s = bv.rms_norm(x, w, r)
    want = bv.rms_norm(x.contiguous(), w, r.contiguous())
    assert torch.equal(y, want[0]) and torch.equal(s, want[1])
    dx, dw = bv.rms_norm_backward(r, x, w, big[:, 2, :200])
    wx, ww = bv.rms_norm_backward(r.contiguous(), x.contiguous(), w,
                                  big[:, 2, :200].contiguous())
    # a row that cannot be read in vectors is summed in another order
    close(dx, wx.double(), 600 * E * wx.double().abs() + 1e-5)
    close(dw, ww.double(), 600 * E * ww.double().abs() + 1e-5)
    grid = rnd(2, 5, 7, 64, dt=BF16)
    assert bv.rms_norm(grid, rnd(64)).shape == grid.shape
    q, scale = bv.rms_norm_e4m3(grid, rnd(64))
    assert q.shape == grid.shape and scale.shape == (2, 5, 7)
    e = torch.empty(0, 64, device="cuda", dtype=BF16)
    assert bv.rms_norm(e, rnd(64)).shape == (0, 64)
    dx, dw = bv.rms_norm_backward(e, e, rnd(64))
    assert dx.shape == (0, 64) and (dw == 0).all()


# ------------------------------------------------------------------- products

SHAPES = [(1, 8, 8), (1, 64, 128), (2, 72, 136), (3, 1, 1), (5, 17, 9), (16, 256, 640),
          (17, 130, 200), (33, 264, 96), (64, 512, 64), (65, 64, 250), (127, 96, 128),
          (128, 128, 576), (129, 200, 264), (257, 65, 129), (300, 576, 520), (511, 40, 24),
          (520, 328, 1032)]


@pytest.mark.parametrize("T,K,N", SHAPES)
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("act,bias,res", [("none", False, False), ("silu", True, True)])
def test_linear(T, K, N, dt, act, bias, res):
    x, w = rnd(T, K, dt=dt), rnd(N, K, dt=dt, scale=K ** -0.5, seed=1)
    b = rnd(N, seed=2) if bias else None
    r = rnd(T, N, dt=dt, seed=3) if res else None
    y, z = bv.linear(x, w, b, act=act, residual=r, save=True)
    ref, tol = product(x, w)
    if bias:
        ref = ref + b.double()
    close(z, ref, tol + 4 * E * ref.abs(), "z")
    val = ACTS[act][0](ref) + (r.double() if res else 0)
    close(y, val, 1.13 * tol + 16 * E * (ref.abs() + val.abs() + 1), "y")
    assert torch.equal(bv.linear(x, w, b, act=act, residual=r), y)


@pytest.mark.parametrize("T,K,N", [(129, 1536, 200), (200, 2048, 64), (130, 4096, 520),
                                   (300, 1100, 72), (129, 4096, 4096)])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_linear_long_sums(T, K, N, dt):
    """Few output tiles and a long K, where K is shared out over work items and
    the shares are joined by a second kernel -- unless there is an epilogue."""
    x, w, b = rnd(T, K, dt=dt), rnd(N, K, dt=dt, scale=K ** -0.5, seed=1), rnd(N, seed=2)
    ref, tol = product(x, w)
    for out in (None, F32):
        for _ in range(6):  # one after the other, each while the last one ends
            y = bv.linear(x, w, out_dtype=out)
        close(y, ref, tol)
        close(bv.linear(x, w, b, out_dtype=out), ref + b.double(), tol + 4 * E * ref.abs())
    bv.blocks_status()


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("out", [None, F32])
@pytest.mark.parametrize("T", [9, 200])
def test_linear_activations(act, out, T):
    x, w = rnd(T, 64, dt=F16, scale=2), rnd(96, 64, dt=F16, scale=0.2, seed=1)
    y = bv.linear(x, w, act=act, out_dtype=out)
    ref, tol = product(x, w)
    val = ACTS[act][0](ref)
    assert y.dtype == (out or F16)
    close(y, val, 1.13 * tol + 32 * E * (ref.abs() + 1))


@pytest.mark.parametrize("T,K,N", [(129, 64, 8), (200, 72, 200), (300, 128, 584), (513, 200, 264),
                                   (140, 65, 131)])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "tanh"])
@pytest.mark.parametrize("dt,out", [(BF16, None), (F16, None), (F16, F32)])
def test_linear_bias_activation_edges(T, K, N, act, dt, out):
    """A bias and an activation without a residual, output widths that end inside a tile's
    store, with and without the pre-activation kept."""
    x, w = rnd(T, K, dt=dt), rnd(N, K, dt=dt, scale=K ** -0.5, seed=1)
    b = rnd(N, seed=2)
    ref, tol = product(x, w)
    ref = ref + b.double()
    val = ACTS[act][0](ref)
    bound = 1.13 * tol + 16 * E * (ref.abs() + val.abs() + 1)
    close(bv.linear(x, w, b, act=act, out_dtype=out), val, bound)
    close(bv.linear(x, w, b, act=act, out_dtype=out, save=True)[0], val, bound)


def quantized(n, k, seed, scale=1.0):
    q, s = bv.pack_weight_e4m3(rnd(n, k, scale=scale, seed=seed))
    return q, s


@pytest.mark.parametrize("T,K,N", SHAPES)
@pytest.mark.parametrize("out", [BF16, F16, F32])
def test_linear_e4m3(T, K, N, out):
    (x, xs), (w, ws) = quantized(T, K, 0), quantized(N, K, 1, K ** -0.5)
    b, r = rnd(N, seed=2), rnd(T, N, dt=out, seed=3)
    y = bv.linear(x, w, b, act="gelu", residual=r, x_scale=xs, w_scale=ws, out_dtype=out)
    ref, tol = product(x, w, xs, ws)
    ref = ref + b.double()
    val = ACTS["gelu"][0](ref) + r.double()
    close(y, val, 1.13 * tol + 16 * E * (ref.abs() + val.abs() + 1))


@pytest.mark.parametrize("T,K,F", SHAPES)
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_linear(T, K, F, dt, act):
    x = rnd(T, K, dt=dt)
    wg, wu = (rnd(F, K, dt=dt, scale=K ** -0.5, seed=s) for s in (1, 2))
    h, g, u = bv.gated_linear(x, wg, wu, act=act, save=True)
    rg, tg = product(x, wg)
    ru, tu = product(x, wu)
    close(g, rg, tg, "g")
    close(u, ru, tu, "u")
    a = ACTS[act][0](rg)
    tol = 1.13 * tg * (ru.abs() + tu) + a.abs() * tu + 16 * E * (rg.abs() + 1) * ru.abs()
    close(h, a * ru, tol, "h")
    assert torch.equal(bv.gated_linear(x, wg, wu, act=act), h)


@pytest.mark.parametrize("act", ["relu", "sigmoid", "tanh"])
@pytest.mark.parametrize("T", [3, 150])
def test_gated_activations(act, T):
    x, wg, wu = rnd(T, 72, dt=F16), rnd(88, 72, dt=F16, scale=.2), rnd(88, 72, dt=F16, scale=.2,
                                                                       seed=1)
    (rg, tg), (ru, tu) = product(x, wg), product(x, wu)
    a = ACTS[act][0](rg)
    close(bv.gated_linear(x, wg, wu, act=act), a * ru,
          1.13 * tg * (ru.abs() + tu) + a.abs() * tu + 16 * E * (rg.abs() + 1) * ru.abs())


@pytest.mark.parametrize("T,K,F", SHAPES)
@pytest.mark.parametrize("out", [BF16, F32])
def test_gated_linear_e4m3(T, K, F, out):
    (x, xs), (wg, gs), (wu, us) = (quantized(T, K, 0), quantized(F, K, 1, K ** -0.5),
                                   quantized(F, K, 2, K ** -0.5))
    h = bv.gated_linear(x, wg, wu, x_scale=xs, gate_scale=gs, up_scale=us, out_dtype=out)
    (rg, tg), (ru, tu) = product(x, wg, xs, gs), product(x, wu, xs, us)
    a = ACTS["silu"][0](rg)
    tol = 1.13 * tg * (ru.abs() + tu) + a.abs() * tu + 16 * E * (rg.abs() + 1) * ru.abs()
    close(h, a * ru, tol)


def grads(dz, w, x, u):
    """dx, dw of 16-bit dz (rounded: u) and their bounds."""
    a, b, c = dz.double(), w.double(), x.double()
    dx, dw = a @ b, a.T @ c
    sx, sw = a.abs() @ b.abs(), a.abs().T @ c.abs()
    nx, nw = (w.shape[0] + 4) * 2 * E, (x.shape[0] + 4) * 2 * E
    return dx, (nx + u) * sx, dw, (nw + u) * sw


@pytest.mark.parametrize("T,K,N", SHAPES)
@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_linear_backward(T, K, N, dt, act):
    x, w, dy = rnd(T, K, dt=dt), rnd(N, K, dt=dt, scale=K ** -0.5, seed=1), rnd(T, N, dt=dt, seed=2)
    z = rnd(T, N, dt=dt, seed=3) if act != "none" else None
    dx, dw, db = bv.linear_backward(dy, x, w, z, act=act, bias=True)
    dz = dy.double() * (ACTS[act][1](z.double()) if z is not None else 1)
    u = half(dt) + 16 * E if act != "none" else 0.0
    # fp16: what falls below the normal range is off by its smallest step's half
    small = torch.finfo(dt).tiny * half(dt) * 2 if act != "none" else 0.0
    rx, tx, rw, tw = grads(dz, w, x, u)
    close(dx, rx, tx + small * w.double().abs().sum(0), "dx")
    close(dw, rw, tw + small * x.double().abs().sum(0), "dw")
    assert db.dtype == F32
    close(db, dz.sum(0), (T + 32) * E * dz.abs().sum(0) + 16 * E * dy.double().abs().sum(0), "db")
    dx2, dw2, db2 = bv.linear_backward(dy, x, w, z, act=act, bias=True)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2) and torch.equal(db, db2)


@pytest.mark.parametrize("act", list(ACTS))
def test_linear_backward_activations(act):
    T, K, N = 70, 48, 56
    x, w, dy = rnd(T, K, dt=F16), rnd(N, K, dt=F16, seed=1), rnd(T, N, dt=F16, seed=2)
    z = rnd(T, N, dt=F16, scale=3, seed=3) if act != "none" else None
    _, _, db = bv.linear_backward(dy, x, w, z, act=act, bias=True, dx=False, dw=False)
    dz = dy.double() * (ACTS[act][1](z.double()) if z is not None else 1)
    close(db, dz.sum(0), (T + 32) * E * dz.abs().sum(0) + 32 * E * dy.double().abs().sum(0))


@pytest.mark.parametrize("T,K,F", SHAPES)
@pytest.mark.parametrize("dt,act", [(BF16, "silu"), (F16, "gelu"), (F16, "relu")])
def test_gated_backward(T, K, F, dt, act):
    x = rnd(T, K, dt=dt)
    wg, wu = (rnd(F, K, dt=dt, scale=K ** -0.5, seed=s) for s in (1, 2))
    dh, g, u = (rnd(T, F, dt=dt, seed=s) for s in (3, 4, 5))
    dx, dwg, dwu = bv.gated_linear_backward(dh, x, wg, wu, g, u, act=act)
    f, d = ACTS[act]
    dg, du = dh.double() * u.double() * d(g.double()), dh.double() * f(g.double())
    # the derivative is good to 16 e of 1 + |g|, whatever its own size
    eps = half(dt)
    fine = 16 * E * dh.double().abs() * (1 + u.double().abs()) * (1 + g.double().abs())
    small = torch.finfo(dt).tiny * eps * 2
    gx, tgx, gw, tgw = grads(dg, wg, x, eps)
    ux, tux, uw, tuw = grads(du, wu, x, eps)
    off_x = (fine + small) @ (wg.double().abs() + wu.double().abs())
    off_w = (fine + small).T @ x.double().abs()
    close(dx, gx + ux, tgx + tux + off_x + 2 * E * F * (tgx + tux) / eps, "dx")
    close(dwg, gw, tgw + off_w, "dw_gate")
    close(dwu, uw, tuw + off_w, "dw_up")
    again = bv.gated_linear_backward(dh, x, wg, wu, g, u, act=act)
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, dwg, dwu)))


def test_backward_against_differences():
    """The gradients of both products along a direction, against central
    differences of the forward formula in 64 bits: the fp16 gradients are off by
    2^-11 of each term, which add up like their absolute values at most."""
    T, K, F = 20, 24, 40
    x, wg, wu, dh = (rnd(*s, dt=F16, seed=i) for i, s in
                     enumerate([(T, K), (F, K), (F, K), (T, F)]))
    v = [rnd(*t.shape, seed=9 + i).double() for i, t in enumerate((x, wg, wu))]
    g, u = (product(x, w)[0].to(F16) for w in (wg, wu))
    # the backward pass takes the rounded projections: so does the formula here
    off_g, off_u = g.double() - product(x, wg)[0], u.double() - product(x, wu)[0]

    def loss(h):
        a, b, c = (t.double() + h * d for t, d in zip((x, wg, wu), v))
        return (dh.double() * ACTS["silu"][0](a @ b.T + off_g) * (a @ c.T + off_u)).sum()

    want = (loss(1e-5) - loss(-1e-5)) / 2e-5
    got = bv.gated_linear_backward(dh, x, wg, wu, g, u)
    terms = [p.double() * d for p, d in zip(got, v)]
    dg = (dh.double() * u.double() * ACTS["silu"][1](g.double())).abs()
    du = (dh.double() * ACTS["silu"][0](g.double())).abs()
    size = ((dg @ wg.double().abs() + du @ wu.double().abs()) * v[0].abs()).sum() \
        + ((dg.T @ x.double().abs()) * v[1].abs()).sum() \
        + ((du.T @ x.double().abs()) * v[2].abs()).sum()
    assert abs(sum(t.sum() for t in terms) - want) <= 2.1 * 2.0 ** -11 * size + 1e-6 * abs(want)

    N = 32
    w, dy = rnd(N, K, dt=F16, seed=20), rnd(T, N, dt=F16, seed=21)
    b, z0 = rnd(N, seed=22), None
    z0 = (product(x, w)[0] + b.double())
    z = z0.to(F16)
    vb = rnd(N, seed=23).double()
    vw = rnd(N, K, seed=24).double()

    def loss2(h):
        zz = (x.double() + h * v[0]) @ (w.double() + h * vw).T + b.double() + h * vb
        return (dy.double() * ACTS["gelu"][0](zz + z.double() - z0)).sum()

    want = (loss2(1e-5) - loss2(-1e-5)) / 2e-5
    dx, dw, db = bv.linear_backward(dy, x, w, z, act="gelu", bias=True)
    got = (dx.double() * v[0]).sum() + (dw.double() * vw).sum() + (db.double() * vb).sum()
    dz = (dy.double() * ACTS["gelu"][1](z.double())).abs()
    size = ((dz @ w.double().abs()) * v[0].abs()).sum() + ((dz.T @ x.double().abs()) * vw.abs()).sum()
    assert abs(got - want) <= 2.1 * 2.0 ** -11 * size + 1e-6 * (abs(want) + 1)


def test_partial_gradients():
    T, K, N = 40, 64, 72
    x, w, dy, z = rnd(T, K, dt=BF16), rnd(N, K, dt=BF16), rnd(T, N, dt=BF16), rnd(T, N, dt=BF16)
    full = bv.linear_backward(dy, x, w, z, act="silu", bias=True)
    assert bv.linear_backward(dy, x, w, z, act="silu", dw=False)[1:] == (None, None)
    assert torch.equal(bv.linear_backward(dy, x, w, z, act="silu", dw=False)[0], full[0])
    assert torch.equal(bv.linear_backward(dy, x, w, z, act="silu", dx=False)[1], full[1])
    gx, gg, gu = bv.gated_linear_backward(dy, x, w, w, z, dy)
    assert torch.equal(bv.gated_linear_backward(dy, x, w, w, z, dy, dw=False)[0], gx)
    p, q, r = bv.gated_linear_backward(dy, x, w, w, z, dy, dx=False)
    assert p is None and torch.equal(q, gg) and torch.equal(r, gu)


@pytest.mark.parametrize("dt", [BF16, F16])
def test_products_on_strided_and_misaligned_rows(dt):
    """Column ranges of wider tensors, at starts and pitches on and off 16 bytes."""
    for T, K, N, off, pitch in ((50, 64, 96, 8, 128), (50, 64, 96, 3, 131), (140, 50, 70, 1, 77),
                                (3, 120, 130, 5, 129), (200, 72, 64, 0, 73)):
        wide = [rnd(n, off + c + pitch, dt=dt, seed=s)[:, off:off + c] for s, (n, c) in
                enumerate(((T, K), (N, K), (N, K), (T, N), (T, N)))]
        flat = [t.contiguous() for t in wide]
        x, w, w2, r, z = wide
        X, W, W2, R, Z = flat
        same = lambda a, b: all(torch.equal(p, q) for p, q in zip(a, b))  # noqa: E731
        assert torch.equal(bv.linear(x, w, residual=r), bv.linear(X, W, residual=R))
        assert torch.equal(bv.gated_linear(x, w, w2), bv.gated_linear(X, W, W2))
        assert same(bv.linear_backward(r, x, w, z, act="tanh", bias=True),
                    bv.linear_backward(R, X, W, Z, act="tanh", bias=True))
        assert same(bv.gated_linear_backward(r, x, w, w2, z, r),
                    bv.gated_linear_backward(R, X, W, W2, Z, R))


def test_leading_axes_empty_and_single_rows():
    w, b = rnd(40, 64, dt=BF16), rnd(40)
    grid = rnd(2, 3, 5, 64, dt=BF16)
    y = bv.linear(grid, w, b)
    assert y.shape == (2, 3, 5, 40)
    assert torch.equal(y.reshape(30, 40), bv.linear(grid.reshape(30, 64), w, b))
    one = bv.linear(grid[0, 0, 0], w, b)
    assert one.shape == (40,)
    e = torch.empty(0, 64, device="cuda", dtype=BF16)
    assert bv.linear(e, w, b).shape == (0, 40)
    assert bv.gated_linear(e, w, w).shape == (0, 40)
    d = torch.empty(0, 40, device="cuda", dtype=BF16)
    dx, dw, db = bv.linear_backward(d, e, w, bias=True)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()
    dx, dg, du = bv.gated_linear_backward(d, e, w, w, d, d)
    assert (dg == 0).all() and (du == 0).all()


def test_infinities_and_nan_stay_in_their_rows():
    T, K, N = 140, 96, 72
    x, w = rnd(T, K, dt=BF16), rnd(N, K, dt=BF16)
    clean = bv.linear(x, w, act="relu")
    cleang = bv.gated_linear(x, w, w)
    bad = x.clone()
    bad[17, 3] = float("nan")
    bad[130, 90] = float("inf")
    y, h = bv.linear(bad, w, act="relu"), bv.gated_linear(bad, w, w)
    rows = [t for t in range(T) if t not in (17, 130)]
    assert torch.equal(y[rows], clean[rows]) and torch.equal(h[rows], cleang[rows])
    assert y[17].isnan().all() and h[17].isnan().all()
    want = torch.relu((bad[130:131].double() @ w.double().T))
    assert torch.equal(y[130].double().isinf(), want[0].isinf())
    wb = w.clone()
    wb[5] = float("nan")
    y = bv.linear(x[:3], wb)
    assert y[:, 5].isnan().all() and not y[:, 6:].isnan().any() and not y[:, :5].isnan().any()


def test_outputs_outside_their_rows_are_left(monkeypatch):
    """The C entry on row strides wider than the rows: what lies between and
    behind the rows keeps its bytes."""
    for T, K, N, ld in ((5, 64, 40, 48), (130, 72, 100, 111), (300, 64, 130, 136)):
        x, w = rnd(T, K, dt=F16), rnd(N, K, dt=F16)
        y = torch.full((T + 2, ld), 7.0, device="cuda", dtype=F16)
        a = B.LinearArgs(x=x.data_ptr(), w=w.data_ptr(), y=y[1:].data_ptr(), ldx=K, ldw=K, ldy=ld,
                         T=T, K=K, N=N, in_type=1, out_type=1, act=0)
        need = B.blocks_lib.bvml_linear_workspace_bytes(ctypes.byref(a))
        ws = torch.empty(max(need, 1), device="cuda", dtype=torch.uint8)
        rc = B.blocks_lib.bvml_linear(ctypes.byref(a), ws.data_ptr(), need,
                                      torch.cuda.current_stream().cuda_stream)
        assert rc == 0, B.blocks_lib.bvml_blocks_last_error()
        assert torch.equal(y[1:T + 1, :N], bv.linear(x, w))
        assert (y[0] == 7).all() and (y[T + 1] == 7).all() and (y[:, N:] == 7).all()


def block(x, p, dt8=False):
    """A pre-norm feed-forward block as a user's program writes it; returns what
    its backward pass needs too."""
    if dt8:
        q, s = bv.rms_norm_e4m3(x, p["n"])
        h = bv.gated_linear(q, p["wg8"], p["wu8"], x_scale=s, gate_scale=p["gs"],
                            up_scale=p["us"], out_dtype=x.dtype)
        return bv.linear(h, p["wd"], p["b"], residual=x)
    n = bv.rms_norm(x, p["n"])
    h, g, u = bv.gated_linear(n, p["wg"], p["wu"], save=True)
    return bv.linear(h, p["wd"], p["b"], residual=x), (n, h, g, u)


def block_backward(dy, x, p, kept):
    n, h, g, u = kept
    dh, dwd, db = bv.linear_backward(dy, h, p["wd"], bias=True)
    dn, dwg, dwu = bv.gated_linear_backward(dh, n, p["wg"], p["wu"], g, u)
    dx, dnw = bv.rms_norm_backward(dn, x, p["n"], dy)
    return dict(x=dx, n=dnw, wg=dwg, wu=dwu, wd=dwd, b=db)


def block_params(K, F, dt):
    p = dict(n=rnd(K) * 0.2 + 1, wg=rnd(F, K, dt=dt, scale=K ** -.5),
             wu=rnd(F, K, dt=dt, scale=K ** -.5, seed=1),
             wd=rnd(K, F, dt=dt, scale=F ** -.5, seed=2), b=rnd(K, seed=3) * 0.1)
    p["wg8"], p["gs"] = bv.pack_weight_e4m3(p["wg"])
    p["wu8"], p["us"] = bv.pack_weight_e4m3(p["wu"])
    return p


def block_ref(x, p):
    n = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * p["n"]
    g = n @ p["wg"].T
    return (g * torch.sigmoid(g) * (n @ p["wu"].T)) @ p["wd"].T + p["b"] + x


@pytest.mark.parametrize("T", [1, 6, 150])
def test_block_forward_and_backward(T):
    """Norm, gated projections and the projection back, as used together:
    against autograd of the formula in 64 bits. Every intermediate is rounded to
    16 bits (six roundings on the longest path): each entry is held to the
    norm of its tensor times 8 half steps."""
    K, F, dt = 128, 320, F16
    p, x, dy = block_params(K, F, dt), rnd(T, K, dt=dt, seed=7), rnd(T, K, dt=dt, seed=8)
    y, kept = block(x, p)
    got = block_backward(dy, x, p, kept)
    leaves = {k: p[k].double().requires_grad_() for k in ("n", "wg", "wu", "wd", "b")}
    x64 = x.double().requires_grad_()
    ref = block_ref(x64, leaves)
    ref.backward(dy.double())
    rms = lambda t: t.double().square().mean().sqrt()  # noqa: E731
    assert rms(y - ref) <= 8 * half(dt) * rms(ref)
    for k, t in {**leaves, "x": x64}.items():
        assert rms(got[k] - t.grad) <= 8 * half(dt) * rms(t.grad), k


@pytest.mark.parametrize("T", [1, 19, 200])
def test_block_in_8_bits(T):
    """The serving form: 8-bit rows and weights against the same values widened."""
    K, F = 256, 384
    p, x = block_params(K, F, BF16), rnd(T, K, dt=BF16, seed=7)
    y = block(x, p, dt8=True)
    q, s = bv.rms_norm_e4m3(x, p["n"])
    n = q.double() * s.double()[:, None]
    g, u = ((n @ (p[w].double() * p[c].double()[:, None]).T) for w, c in (("wg8", "gs"),
                                                                        ("wu8", "us")))
    ref = (g * torch.sigmoid(g) * u) @ p["wd"].double().T + p["b"].double() + x.double()
    d = (y.double() - ref).abs()
    # h is rounded to bf16 once, the result once
    h = (g * torch.sigmoid(g) * u).abs() @ p["wd"].double().abs().T
    assert (d <= half(BF16) * (ref.abs() + 1.01 * h) + 1e-5).all()


def test_streams_and_graphs():
    """The block on a side stream, and captured and replayed with new inputs;
    two graphs with workspaces of their own replayed on two streams."""
    K, F, dt = 128, 200, BF16
    p = block_params(K, F, dt)
    p["wd"] = rnd(K, F + 1, dt=dt)[:, 1:]  # misaligned rows: laid out in a workspace
    xs = [rnd(70, K, dt=dt, seed=s) for s in range(4)]
    dys = [rnd(70, K, dt=dt, seed=10 + s) for s in range(4)]

    def step(x, dy):
        y, kept = block(x, p)
        return y, block_backward(dy, x, p, kept)

    want = [step(x, dy) for x, dy in zip(xs, dys)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step(xs[0], dys[0])
    side.synchronize()
    same = lambda a, b: torch.equal(a[0], b[0]) and all(  # noqa: E731
        torch.equal(a[1][k], b[1][k]) for k in a[1])
    assert same(got, want[0])
    graphs = []
    for i in range(2):
        sx, sdy = xs[i].clone(), dys[i].clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(sx, sdy)
        graphs.append((g, sx, sdy, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for base in (0, 2):
        torch.cuda.synchronize()
        for i, (g, sx, sdy, out) in enumerate(graphs):
            sx.copy_(xs[base + i])
            sdy.copy_(dys[base + i])
        torch.cuda.synchronize()
        for rep in range(5):
            for (g, *_), st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for i, (_, _, _, out) in enumerate(graphs):
            assert same(out, want[base + i])
    bv.blocks_status()


def test_python_argument_errors():
    x, w = rnd(4, 64, dt=BF16), rnd(8, 64, dt=BF16)
    with pytest.raises(RuntimeError, match="weight has 32 columns"):
        bv.linear(x, w[:, :32])
    with pytest.raises(RuntimeError, match="weight must be"):
        bv.linear(x, w.half())
    with pytest.raises(RuntimeError, match="last axis must be contiguous"):
        bv.linear(x.T.contiguous().T, w)
    with pytest.raises(RuntimeError, match="rows overlap"):
        bv.linear(x[:1].expand(4, 64), w)
    with pytest.raises(RuntimeError, match="evenly spaced"):
        bv.linear(rnd(4, 6, 64, dt=BF16)[:, :3], w)
    with pytest.raises(RuntimeError, match="inputs must be fp16"):
        bv.linear(x.float(), w.float())
    with pytest.raises(RuntimeError, match="output must be"):
        bv.linear(x, w, out_dtype=F16)
    with pytest.raises(RuntimeError, match="unknown activation"):
        bv.linear(x, w, act="swish")
    with pytest.raises(RuntimeError, match="bias must be"):
        bv.linear(x, w, rnd(8, dt=BF16))
    with pytest.raises(RuntimeError, match="bias has 7"):
        bv.linear(x, w, rnd(7))
    with pytest.raises(RuntimeError, match="need their scales"):
        bv.linear(x.to(E4M3), w.to(E4M3))
    with pytest.raises(RuntimeError, match="scales belong"):
        bv.linear(x, w, x_scale=rnd(4), w_scale=rnd(8))
    with pytest.raises(RuntimeError, match="no autograd"):
        bv.linear(x, w.clone().requires_grad_())
    with torch.no_grad():
        bv.linear(x, w.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="z belongs"):
        bv.linear_backward(rnd(4, 8, dt=BF16), x, w, act="silu")
    with pytest.raises(RuntimeError, match="unsupported storage"):
        bv.rms_norm(x.double(), rnd(64))
    with pytest.raises(RuntimeError, match="weight must be"):
        bv.rms_norm(x, rnd(64, dt=F16))
    with pytest.raises(RuntimeError, match="x's shape"):
        bv.rms_norm(x, rnd(64), x[:2])
    with pytest.raises(RuntimeError, match="share a device"):
        bv.linear(x, w.cpu())


def _c_call(lib, name, args):
    """A C entry point of `lib` with a workspace of its own."""
    fn, size = getattr(lib, name), getattr(lib, name + "_workspace_bytes")
    ref = getattr(B.blocks_lib, name)
    fn.argtypes, fn.restype = ref.argtypes, ref.restype
    size.argtypes, size.restype = ref.argtypes[:1], ctypes.c_size_t
    need = size(ctypes.byref(args))
    ws = torch.empty(max(need, 1), device="cuda", dtype=torch.uint8)
    assert fn(ctypes.byref(args), ws.data_ptr(), need,
              torch.cuda.current_stream().cuda_stream) == 0


@pytest.mark.parametrize("T,K,N", [(1, 8, 8), (16, 256, 640), (128, 136, 72), (129, 2048, 264),
                                   (257, 65, 129), (520, 328, 1032)])
def test_checked_build(T, K, N):
    """The checked build (every TMA copy's coordinate and address tested before it is
    issued) records nothing and computes what the release build does."""
    import os

    path = os.path.join(os.path.dirname(bv.BLOCKS_LIB_PATH), "libbvml_blocks_checked.so")
    checked = ctypes.CDLL(path)
    checked.bvml_blocks_status.argtypes = [ctypes.c_void_p]
    x, w, w2, dy = (rnd(n, c, dt=BF16, seed=s) for s, (n, c) in
                    enumerate(((T, K), (N, K), (N, K), (T, N))))
    outs = {}
    for lib in (B.blocks_lib, checked):
        y, h, g, u = (torch.empty(T, N, device="cuda", dtype=BF16) for _ in range(4))
        dx, dw, dg, du = (torch.empty(n, K, device="cuda", dtype=BF16) for n in (T, N, N, N))
        _c_call(lib, "bvml_linear", B.LinearArgs(
            x=x.data_ptr(), w=w.data_ptr(), y=y.data_ptr(), ldx=K, ldw=K, ldy=N, T=T, K=K, N=N,
            in_type=2, out_type=2, act=0))
        _c_call(lib, "bvml_gated_linear", B.GatedArgs(
            x=x.data_ptr(), w_gate=w.data_ptr(), w_up=w2.data_ptr(), h=h.data_ptr(),
            g=g.data_ptr(), u=u.data_ptr(), ldx=K, ldw_gate=K, ldw_up=K, ldh=N, ldg=N, ldu=N,
            T=T, K=K, F=N, in_type=2, out_type=2, act=4))
        _c_call(lib, "bvml_linear_backward", B.LinearBackwardArgs(
            dy=dy.data_ptr(), z=g.data_ptr(), x=x.data_ptr(), w=w.data_ptr(), dx=dx.data_ptr(),
            dw=dw.data_ptr(), lddy=N, ldz=N, ldx=K, ldw=K, lddx=K, lddw=K, T=T, K=K, N=N, type=2,
            act=5))
        dx2 = torch.empty_like(dx)
        _c_call(lib, "bvml_gated_linear_backward", B.GatedBackwardArgs(
            dh=dy.data_ptr(), g=g.data_ptr(), u=u.data_ptr(), x=x.data_ptr(),
            w_gate=w.data_ptr(), w_up=w2.data_ptr(), dx=dx2.data_ptr(), dw_gate=dg.data_ptr(),
            dw_up=du.data_ptr(), lddh=N, ldg=N, ldu=N, ldx=K, ldw_gate=K, ldw_up=K, lddx=K,
            lddw_gate=K, lddw_up=K, T=T, K=K, F=N, type=2, act=4))
        assert lib.bvml_blocks_status(torch.cuda.current_stream().cuda_stream) == 0
        outs[lib] = (y, h, g, u, dx, dw, dx2, dg, du)
    assert all(torch.equal(p, q) for p, q in zip(outs[B.blocks_lib], outs[checked]))


def test_misaligned_vectors():
    """A bias and scales that start on no 16 bytes, with few and many rows."""
    for T in (7, 150):
        x, w, b = rnd(T, 64, dt=BF16), rnd(96, 64, dt=BF16), rnd(97)
        ref, tol = product(x, w)
        close(bv.linear(x, w, b[1:], act="relu"), torch.relu(ref + b[1:].double()),
              tol + 8 * E * (ref.abs() + 4))
        (q, s), (v, t) = quantized(T, 64, 0), quantized(96, 64, 1)
        t1 = torch.cat([t[:1], t])[1:]
        assert torch.equal(bv.linear(q, v, x_scale=s, w_scale=t1),
                           bv.linear(q, v, x_scale=s, w_scale=t))
        assert torch.equal(bv.gated_linear(q, v, v, x_scale=s, gate_scale=t1, up_scale=t),
                           bv.gated_linear(q, v, v, x_scale=s, gate_scale=t, up_scale=t))


def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: the last rows are what they are alone."""
    T, K, N = 270_000, 8192, 64
    x = torch.empty(T, K, device="cuda", dtype=BF16)
    x[:256] = rnd(256, K, dt=BF16)
    x[256:-300] = 0
    x[-300:] = rnd(300, K, dt=BF16, seed=1)
    w, nw = rnd(N, K, dt=BF16, scale=0.02), rnd(K) + 1
    assert x.numel() > 2 ** 31
    y = bv.linear(x, w)
    # (many rows and few are summed in another order)
    ref, tol = product(x[-300:], w)
    close(y[-300:], ref, tol)
    assert (y[256:-300] == 0).all()
    n = bv.rms_norm(x, nw)
    assert torch.equal(n[-300:], bv.rms_norm(x[-300:], nw))
    assert torch.equal(n[:256], bv.rms_norm(x[:256], nw))
    dx, _ = bv.rms_norm_backward(n, x, nw)
    want = bv.rms_norm_backward(n[-300:], x[-300:], nw)[0]
    assert torch.equal(dx[-300:], want)
    del dx, n
    dy = rnd(T, N, dt=BF16, seed=3)
    dx, _, _ = bv.linear_backward(dy, x, w, dw=False)
    ref = dy[-300:].double() @ w.double()
    close(dx[-300:], ref, (N + 4) * 2 * E * (dy[-300:].double().abs() @ w.double().abs()))
