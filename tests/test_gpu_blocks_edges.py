"""The feed-forward operators at the edges of what their documents allow. Bounds as in
test_gpu_blocks.py."""
import pytest
import torch

import brovisionml_b200 as bv
from brovisionml_b200 import _blocks_capi as B
from test_gpu_blocks import (ACTS, BF16, E, E4M3, F16, F32, close, grads, product, quantized,
                             rnd)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lead", [(0,), (2, 0), (0, 3)])
def test_empty_batches_in_8_bits(lead):
    """The 8-bit chain on no rows: norm, gated product, product."""
    x = torch.empty(*lead, 64, device="cuda", dtype=BF16)
    q, scale = bv.rms_norm_e4m3(x, rnd(64))
    assert q.shape == x.shape and q.dtype == E4M3 and scale.shape == lead
    (w, ws), (v, vs) = quantized(40, 64, 0), quantized(40, 64, 1)
    h = bv.gated_linear(q, w, v, x_scale=scale, gate_scale=ws, up_scale=vs)
    assert h.shape == (*lead, 40) and h.dtype == BF16
    y, z = bv.linear(q, w, rnd(40), x_scale=scale, w_scale=ws, out_dtype=F32, save=True)
    assert y.shape == z.shape == (*lead, 40) and y.dtype == F32


@pytest.mark.parametrize("K", [64, 65, 640, 4096, 16400])
@pytest.mark.parametrize("dt", [BF16, F32])
def test_rms_norm_e4m3_of_small_rows(K, dt):
    """Rows near and below the smallest normal numbers: finite where the norm is, as the
    formula has them (their |s w| rounded to 32 bits: half of 2^-149 at least), zeros below
    2^-110."""
    sizes = (1e-30, 7e-31, 1e-33, 1e-35, 1.4e-36, 1.2e-36, 1e-36, 8e-37, 6e-37, 1e-37, 2e-39)
    for eps in (1e-6, 1e-12):
        x = rnd(len(sizes), K)
        x = (x / x.abs().amax(1, keepdim=True) * torch.tensor(sizes, device="cuda")[:, None]).to(dt)
        w = rnd(K, seed=1).abs() * 0.1 + 0.9
        q, scale = bv.rms_norm_e4m3(x, w, eps=eps)
        y = x.double() * w.double() * (x.double().square().mean(1, keepdim=True) + eps).rsqrt()
        top = y.abs().amax(1)
        zero, some = top < 2.0 ** -110 * (1 - 1e-3), top > 2.0 ** -110 * (1 + 1e-3)
        assert some.sum() > 3
        assert (scale[zero] == 1).all() and (q[zero].float() == 0).all()
        y, top, q, scale = y[some], top[some], q[some].double(), scale[some].double()
        # |s w| is off by half a step, which below 2^-126 is 2^-150, times the root
        fine = (K / 2 + 16) * E
        step = 2.0 ** -150 * eps ** -0.5
        assert ((scale - top / 448).abs() <= fine * top / 448 + step / 448).all()
        off = ((q * scale[:, None] - y).abs()
               - (2.0 ** -4 + 2 * fine) * y.abs() - scale[:, None] * 2.0 ** -10 - 2 * step)
        assert (off <= 0).all(), off.max()
    z = torch.zeros(2, K, device="cuda", dtype=dt)
    q, scale = bv.rms_norm_e4m3(z, w, eps=0.0)
    assert scale.isnan().all() and q.float().isnan().all()  # 0 / 0


@pytest.mark.parametrize("K", [64, 65, 128, 200, 500, 1000, 1001, 4096, 16400])
def test_rms_norm_e4m3_of_equal_largest_products(K):
    """Two elements whose products with their weights are equal in 32 bits and not beyond:
    the larger one gives the row's scale for all of the row, wherever the two stand. The
    values beside them lie next to rounding borders of the 8 bits (17, 23, 272, ...)."""
    h = float.fromhex
    tops = [(h("0x1.63c556p+0"), h("0x1.432a7p+0")), (h("0x1.48dfd4p+0"), h("0x1.5d986ep+0"))]
    assert len({float(torch.tensor(a) * torch.tensor(b)) for a, b in tops}) == 1
    beside = [h(v) for v in ("0x1.10ad04p-4", "0x1.70ea14p-4", "0x1.d12724p-4", "0x1.10ad04p+0",
                             "0x1.70ea14p+0")]
    most = max(a * b for a, b in tops)
    want = torch.tensor([v * 448 / most for v in beside]).to(E4M3).float()
    x = torch.zeros(6, K, device="cuda")
    w = torch.ones(6, K, device="cuda")
    at = [(0, 40, 1), (1, 63, 2), (K - 1, 7, K // 2), (K // 2, K - 2, 5), (8, 9, 17), (33, 2, 44)]
    for t, (i, j, k) in enumerate(at):
        x[t, i], w[t, i] = tops[t % 2]
        x[t, j], w[t, j] = tops[1 - t % 2]
        free = [p for p in range(K) if p not in (i, j)]
        for n, p in enumerate(free):
            x[t, p] = beside[n % 5]
        q, scale = bv.rms_norm_e4m3(x[t:t + 1], w[t])
        got = q[0, free].float().cpu()
        assert torch.equal(got, want.repeat(K // 5 + 1)[:len(free)]), t
        assert (q[0, [i, j]].float() == 448).all()


@pytest.mark.parametrize("act", ["sigmoid", "tanh"])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_derivatives_far_from_zero(act, dt):
    """Derivatives that go to zero keep their figures: e^-|z| (e^-2|z|) from a rounded
    argument and the hardware's 2^x and 1 / x are good to (4 |z| + 16) 2^-24 together, and
    below 2^-126 flush to zero. Alone (the bias gradient of one row) and through the gate."""
    z = torch.cat([torch.linspace(-60, 60, 961), torch.tensor([3e38, -3e38])]).cuda().to(dt)
    z[0], z[1] = float("inf"), float("-inf")
    N = z.numel()
    one = torch.ones(1, N, device="cuda", dtype=dt)
    x, w = torch.ones(1, 8, device="cuda", dtype=dt), torch.zeros(N, 8, device="cuda", dtype=dt)
    _, _, db = bv.linear_backward(one, x, w, z[None], act=act, bias=True, dx=False, dw=False)
    v = z.double().abs()
    a = torch.exp(-v if act == "sigmoid" else -2 * v)
    ref = a / (1 + a) ** 2 * (1 if act == "sigmoid" else 4)
    rel = torch.where(v.isinf(), torch.zeros_like(v), (4 * v + 16) * E * ref)
    assert ((db.double() - ref).abs() <= rel + 2.0 ** -123).all()
    x[0, 1:] = 0  # dw_gate[:, 0] = dg = dh u act'(g)
    _, dg, du = bv.gated_linear_backward(one, x, w, w, z[None], one, act=act, dx=False)
    small = torch.finfo(dt).tiny * torch.finfo(dt).eps  # the smallest step, halved twice
    assert ((dg[:, 0].double() - ref).abs()
            <= rel + (ref + rel) * torch.finfo(dt).eps / 2 + small / 2 + 2.0 ** -123).all()
    f = torch.sigmoid(z.double()) if act == "sigmoid" else torch.tanh(z.double())
    assert ((du[:, 0].double() - f).abs() <= f.abs() * (torch.finfo(dt).eps / 2 + 200 * E)
            + small / 2 + 2.0 ** -123).all()
    nan = torch.full_like(one, float("nan"))
    _, _, db = bv.linear_backward(one, x, w, nan, act=act, bias=True, dx=False, dw=False)
    assert db.isnan().all()


def _waits(case):
    """(a call and its outputs) for a kernel of the products."""
    T, K, N = case["size"]
    x, w, w2, dy = (rnd(*s, dt=BF16, scale=0.1, seed=i) for i, s in
                    enumerate([(T, K), (N, K), (N, K), (T, N)]))
    if case["op"] == "linear":
        return lambda: (bv.linear(x, w),)
    if case["op"] == "gated":
        return lambda: (bv.gated_linear(x, w, w2),)
    if case["op"] == "backward":
        return lambda: bv.linear_backward(dy, x, w)[:2]
    (q, s), (v, t) = quantized(T, K, 0), quantized(N, K, 1)
    return lambda: (bv.linear(q, v, x_scale=s, w_scale=t),)


@pytest.mark.parametrize("case", [
    dict(op="linear", size=(5, 4096, 1000)),  # few rows, K over a cluster
    dict(op="gated", size=(100, 2048, 600)),
    dict(op="e4m3", size=(60, 4096, 500)),
    dict(op="linear", size=(520, 64, 264)),  # tiles: fewer K steps than the ring holds
    dict(op="linear", size=(520, 2048, 1032)),
    dict(op="linear", size=(200, 4096, 256)),  # shares of K
    dict(op="gated", size=(1300, 320, 4000)),  # several tiles a pair
    dict(op="e4m3", size=(3000, 640, 2600)),
    dict(op="backward", size=(2900, 2900, 264)),
], ids=lambda c: f"{c['op']}-{'x'.join(map(str, c['size']))}")
def test_waits_that_give_up(case):
    """A short limit on the waits between a product's copies, MMAs and epilogue: the call
    ends, the status tells of it, and the next call on the stream is what it was. With one
    attempt the first MMA never finds its operands; with more the waits that give up are
    spread over the kernel, or none does and the result stands."""
    call = _waits(case)
    bv.blocks_status()
    want = call()
    bv.blocks_status()
    limit = B.blocks_lib.bvml_blocks_wait_limit
    for attempts in (1, 2, 3, 5, 9, 17, 33):
        assert limit(attempts) == 4194304
        try:
            got, gave_up = call(), False
            torch.cuda.synchronize()
            try:
                bv.blocks_status()
            except RuntimeError as e:
                assert "pipeline gave up" in str(e)
                gave_up = True
        finally:
            limit(4194304)
        assert gave_up or attempts > 1
        assert gave_up or all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(call(), want)), attempts
        bv.blocks_status()


# More tiles than pairs of SMs (74): every pair takes several, over both accumulators, with
# the ring's state going on from tile to tile.
MANY = [(3000, 200, 2600), (1300, 72, 5000), (20000, 136, 520)]


@pytest.mark.parametrize("T,K,N", MANY)
@pytest.mark.parametrize("dt,out,act,whole", [(BF16, None, "none", True), (F16, F32, "gelu", False),
                                              (E4M3, BF16, "none", True), (E4M3, F32, "silu", False),
                                              (E4M3, F16, "relu", True)])
def test_linear_of_many_tiles(T, K, N, dt, out, act, whole):
    if dt == E4M3:
        (x, xs), (w, ws) = quantized(T, K, 0), quantized(N, K, 1, K ** -0.5)
        ref, tol = product(x, w, xs, ws)
        scales = dict(x_scale=xs, w_scale=ws)
    else:
        x, w, scales = rnd(T, K, dt=dt), rnd(N, K, dt=dt, scale=K ** -0.5, seed=1), {}
        ref, tol = product(x, w)
    b = rnd(N, seed=2)
    r = None if whole else rnd(T, N, dt=out or dt, seed=3)
    y = bv.linear(x, w, b, act=act, residual=r, out_dtype=out, **scales)
    ref = ref + b.double()
    val = ACTS[act][0](ref) + (0 if whole else r.double())
    close(y, val, 1.13 * tol + 16 * E * (ref.abs() + val.abs() + 1))
    assert torch.equal(bv.linear(x, w, b, act=act, residual=r, out_dtype=out, **scales), y)
    bv.blocks_status()


@pytest.mark.parametrize("T,K,F", MANY)
@pytest.mark.parametrize("dt", [BF16, E4M3])
def test_gated_linear_of_many_tiles(T, K, F, dt):
    if dt == E4M3:
        (x, xs), (wg, gs), (wu, us) = (quantized(T, K, 0), quantized(F, K, 1, K ** -0.5),
                                       quantized(F, K, 2, K ** -0.5))
        scales = dict(x_scale=xs, gate_scale=gs, up_scale=us)
        (rg, tg), (ru, tu) = product(x, wg, xs, gs), product(x, wu, xs, us)
    else:
        x, scales = rnd(T, K, dt=dt), {}
        wg, wu = (rnd(F, K, dt=dt, scale=K ** -0.5, seed=s) for s in (1, 2))
        (rg, tg), (ru, tu) = product(x, wg), product(x, wu)
    h, g, u = bv.gated_linear(x, wg, wu, save=True, **scales)
    close(g, rg, tg + 4 * E * rg.abs(), "g")
    close(u, ru, tu + 4 * E * ru.abs(), "u")
    a = ACTS["silu"][0](rg)
    close(h, a * ru, 1.13 * tg * (ru.abs() + tu) + a.abs() * tu + 16 * E * (rg.abs() + 1) * ru.abs())
    assert torch.equal(bv.gated_linear(x, wg, wu, **scales), h)
    bv.blocks_status()


@pytest.mark.parametrize("T,K,N", [(264, 2700, 2700), (2700, 2700, 264), (130, 5000, 1300)])
def test_gradients_of_many_tiles(T, K, N):
    dt = BF16
    x, dy = rnd(T, K, dt=dt), rnd(T, N, dt=dt, seed=2)
    w, w2 = (rnd(N, K, dt=dt, scale=K ** -0.5, seed=s) for s in (1, 3))
    dx, dw, _ = bv.linear_backward(dy, x, w)
    rx, tx, rw, tw = grads(dy, w, x, 0.0)
    close(dx, rx, tx, "dx")
    close(dw, rw, tw, "dw")
    g, u = rnd(T, N, dt=dt, seed=4), rnd(T, N, dt=dt, seed=5)
    dx, dwg, dwu = bv.gated_linear_backward(dy, x, w, w2, g, u, act="relu")
    # relu's dg and du are one product and one selection: rounded to 16 bits once, exact in 32
    dg = torch.where(g > 0, dy.float() * u.float(), 0).to(dt)
    du = torch.where(g > 0, dy.float() * g.float(), 0).to(dt)
    gx, tgx, gw, tgw = grads(dg, w, x, 0.0)
    ux, tux, uw, tuw = grads(du, w2, x, 0.0)
    # one sum over both halves: up to twice either's number of terms
    close(dx, gx + ux, 2 * (tgx + tux), "dx")
    close(dwg, gw, tgw, "dw_gate")
    close(dwu, uw, tuw, "dw_up")
    bv.blocks_status()


@pytest.mark.parametrize("T,K,N", [(130, 1, 1), (300, 3, 2), (520, 2, 7), (140, 1, 300),
                                   (140, 300, 1)])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_many_rows_of_few_features(T, K, N, dt):
    """Widths below a store of 16 bytes on the tile kernels, forward and backward."""
    x, dy = rnd(T, K, dt=dt), rnd(T, N, dt=dt, seed=2)
    w, w2 = rnd(N, K, dt=dt, seed=1), rnd(N, K, dt=dt, seed=3)
    ref, tol = product(x, w)
    close(bv.linear(x, w), ref, tol)
    ru, tu = product(x, w2)
    g, u = bv.gated_linear(x, w, w2, save=True)[1:]
    close(g, ref, tol)
    close(u, ru, tu)
    dx, dw, db = bv.linear_backward(dy, x, w, bias=True)
    rx, tx, rw, tw = grads(dy, w, x, 0.0)
    close(dx, rx, tx)
    close(dw, rw, tw)
    close(db, dy.double().sum(0), (T + 32) * E * dy.double().abs().sum(0))
    (q, s), (v, t) = quantized(T, K, 4), quantized(N, K, 5)
    ref, tol = product(q, v, s, t)
    close(bv.linear(q, v, x_scale=s, w_scale=t, out_dtype=F32), ref, tol + 4 * E * ref.abs())


@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("T", [1, 200])
def test_activations_far_below_zero(act, T):
    """Down to 2^-126 the activations keep their figures (an argument's rounding counts |z|, or
    z^2 with gelu, times 2^-24); below, sigmoid and exp(-z^2 / 2) flush to zero, which is off
    by |z| 2^-126 at most."""
    z = torch.cat([torch.linspace(-110, 0, 881), torch.linspace(-14, -8, 97)]).cuda().to(BF16)
    x = torch.zeros(T, 8, device="cuda", dtype=BF16)
    x[:, 3] = 1
    w = torch.zeros(z.numel(), 8, device="cuda", dtype=BF16)
    w[:, 3] = z
    y = bv.linear(x, w, act=act, out_dtype=F32).double()
    v = z.double()
    ref = {"sigmoid": torch.sigmoid(v), "silu": v * torch.sigmoid(v),
           "gelu": v * torch.special.erfc(-v / 2 ** 0.5) / 2}[act]
    arg = v * v if act == "gelu" else v.abs()
    tol = (4 * arg + 32) * E * ref.abs() + (v.abs() + 1) * 2.0 ** -126 * 1.01
    assert ((y - ref).abs() <= tol).all()
