"""The feed-forward operators and what is measured of them.

``rms_norm`` (with the residual's addition, 16-bit or 8-bit output, and its
backward pass), ``linear`` (a matrix product with bias, activation and
residual, and its backward pass) and ``gated_linear`` (two projections, the
activation and the product, and its backward pass), over rows of features:
pixels of a grid or tokens of a sequence.

Each case names an operator and its sizes: T rows, K input features, N output
features (F = N for the gated operator). ``run`` computes it in plain torch
operations, or, with ``own`` set, by the framework's kernels.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token of a decoding step through a block's first norm, residual stream updated
        dict(name="norm token", op="norm", T=1, K=4096, dtype="bf16", residual=True),
        # the heads' 128 channels of four 720p frames on the 1/8 grid (90 x 160)
        dict(name="norm pixels", op="norm", T=57600, K=128, dtype="fp16", residual=False),
        # a prompt's rows before an 8-bit product, an odd number of them
        dict(name="norm e4m3 prompt", op="norm_e4m3", T=8197, K=4096, dtype="bf16",
             residual=True),
        # a training step's backward pass through the norm, the residual's gradient added
        dict(name="norm backward", op="norm_backward", T=16384, K=2048, dtype="bf16",
             residual=True),
        # one token through the output projection of a block
        dict(name="linear token", op="linear", T=1, K=4096, N=4096, dtype="bf16", act="none",
             bias=True, residual=True),
        # the last layer of the up-mask head as a product: 128 -> 576 channels, four 720p frames
        dict(name="linear pixels", op="linear", T=57600, K=128, N=576, dtype="fp16", act="none",
             bias=True, residual=False),
        # a prompt's rows: the largest product
        dict(name="linear prompt", op="linear", T=8192, K=4096, N=8192, dtype="bf16", act="gelu",
             bias=True, residual=True),
        # a batch of 61 decoding requests, 8-bit rows and weights
        dict(name="linear e4m3 batch", op="linear_e4m3", T=61, K=4096, N=12288, dtype="bf16",
             act="none", bias=False, residual=False),
        # a training step, ragged in every size
        dict(name="linear backward", op="linear_backward", T=4099, K=1544, N=2056, dtype="fp16",
             act="silu", bias=True),
        # a batch of 16 decoding requests through the gated projections
        dict(name="gated batch", op="gated", T=16, K=4096, N=11264, dtype="bf16", act="silu",
             save=False),
        # a training step's forward pass, which keeps both projections for the backward pass
        dict(name="gated forward", op="gated", T=4096, K=4096, N=11264, dtype="bf16", act="silu",
             save=True),
        # the backward pass of a training step, an odd number of rows
        dict(name="gated backward", op="gated_backward", T=8191, K=2048, N=5632, dtype="bf16",
             act="silu"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A feature width: a multiple of 8 as a rule, any number at times."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.2 else max(8, n // 8 * 8)


def draw(rng):
    op = rng.choice(["norm", "norm_e4m3", "norm_backward", "linear", "linear_e4m3",
                     "linear_backward", "gated", "gated_e4m3", "gated_backward"])
    dtype = rng.choice(["bf16", "fp16"])
    if op.startswith("norm"):
        K = _width(rng, 64, 12000)
        T = _log_int(rng, 1, max(1, min(60000, 33_000_000 // K)))
        if op != "norm_e4m3" and rng.random() < 0.2:
            dtype = "fp32"
        return dict(op=op, T=T, K=K, dtype=dtype, residual=rng.random() < 0.6)
    K, N = _width(rng, 64, 8192), _width(rng, 64, 11264)
    passes = {"linear_backward": 2, "gated": 2, "gated_e4m3": 2, "gated_backward": 4}.get(op, 1)
    # at most half the largest listed case's products, and outputs of a modest size
    T = _log_int(rng, 1, max(1, min(60000, int(1.8e11 / (K * N * passes)), 80_000_000 // N,
                                    100_000_000 // K)))
    act = rng.choice(["silu", "gelu", "relu", "sigmoid", "tanh"])
    case = dict(op=op, T=T, K=K, N=N, dtype=dtype, act=act)
    if op.startswith("linear"):
        case["act"] = rng.choice(["none", act])
        case["bias"] = rng.random() < 0.5
        if op != "linear_backward":
            case["residual"] = rng.random() < 0.5
    elif op != "gated_backward":
        case["save"] = rng.random() < 0.3
    return case


def _quantize_rows(w):
    """e4m3 values and one scale a row: w = q * scale."""
    w = w.float()
    scale = w.abs().amax(1) / E4M3_MAX
    q = (w / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]
    T, K, N = case["T"], case["K"], case.get("N", 0)

    def rnd(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)

    def rows():
        # features of a residual stream: unit size, a few channels much larger
        x = torch.randn((T, K), device="cuda", generator=g)
        x[:, :: max(1, K // 7)] *= 6.0
        return x

    op = case["op"]
    s = {"case": case}
    if op.startswith("norm"):
        s["x"] = rows().to(dt)
        # a norm's weights: kept in 32 bits for half the sizes, in the rows' type for the rest
        s["w"] = rnd(K, scale=0.2, dtype=torch.float32 if K % 16 == 0 else dt) + 1.0
        if case["residual"]:
            s["r"] = rnd(T, K, scale=2.0)
        if op == "norm_backward":
            s["dy"] = rnd(T, K)
        return s
    if op.endswith("e4m3"):
        s["x"], s["xs"] = _quantize_rows(rows() + 1e-3)
    else:
        s["x"] = rows().to(dt)
    names = ("wg", "wu") if op.startswith("gated") else ("w",)
    for n in names:
        w = rnd(N, K, scale=K ** -0.5)
        if op.endswith("e4m3"):
            s[n], s[n + "s"] = _quantize_rows(w)
        else:
            s[n] = w
    if op == "gated_backward":
        s["dh"], s["g"], s["u"] = rnd(T, N), rnd(T, N, scale=1.5), rnd(T, N, scale=1.5)
    elif op == "linear_backward":
        s["dy"] = rnd(T, N)
        s["z"] = rnd(T, N, scale=1.5) if case["act"] != "none" else None
    elif op.startswith("linear"):
        s["b"] = rnd(N, scale=0.3, dtype=torch.float32) if case["bias"] else None
        s["r"] = rnd(T, N, scale=2.0) if case["residual"] else None
    return s


# ---------------------------------------------------------------- plain form


def _act(z, name):
    if name == "relu":
        return torch.clamp(z, min=0)
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if name == "tanh":
        return torch.tanh(z)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_grad(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "sigmoid":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 - p)
    if name == "tanh":
        t = torch.tanh(z)
        return 1 - t * t
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    if name == "gelu":
        return (0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
                + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)))
    return torch.ones_like(z)


def _plain(s):
    case = s["case"]
    op, dt = case["op"], TYPES[case["dtype"]]
    if op == "norm":
        t = s["x"].float() + s["r"].float() if "r" in s else s["x"].float()
        y = t * torch.rsqrt(torch.mean(t * t, 1, keepdim=True) + EPS) * s["w"].float()
        return (y.to(dt), t.to(dt)) if "r" in s else y.to(dt)
    if op == "norm_e4m3":
        # in 64 bits: an 8-bit value next to a rounding border goes by the last bits
        t = s["x"].double() + s["r"].double() if "r" in s else s["x"].double()
        y = t * torch.rsqrt(torch.mean(t * t, 1, keepdim=True) + EPS) * s["w"].double()
        scale = y.abs().amax(1) / E4M3_MAX
        q = (y / scale[:, None]).float().clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        return (q, scale.float(), t.to(dt)) if "r" in s else (q, scale.float())
    if op == "norm_backward":
        t, dy, w = s["x"].float(), s["dy"].float(), s["w"].float()
        rstd = torch.rsqrt(torch.mean(t * t, 1, keepdim=True) + EPS)
        n = t * rstd
        dyw = dy * w
        dx = rstd * (dyw - n * torch.mean(dyw * n, 1, keepdim=True))
        if "r" in s:
            dx = dx + s["r"].float()
        return dx.to(dt), torch.sum(dy * n, 0).to(s["w"].dtype)
    if op.endswith("e4m3"):
        x = s["x"].float() * s["xs"][:, None]
    else:
        x = s["x"].float()
    weight = {n: s[n].float() * s[n + "s"][:, None] if n + "s" in s else s[n].float()
              for n in ("w", "wg", "wu") if n in s}
    if op.startswith("linear") and op != "linear_backward":
        z = x @ weight["w"].T
        if s["b"] is not None:
            z = z + s["b"]
        y = _act(z, case["act"])
        if s["r"] is not None:
            y = y + s["r"].float()
        return y.to(dt)
    if op == "linear_backward":
        dz = s["dy"].float()
        if s["z"] is not None:
            dz = dz * _act_grad(s["z"].float(), case["act"])
        out = ((dz @ weight["w"]).to(dt), (dz.T @ x).to(dt))
        return out + (torch.sum(dz, 0),) if case["bias"] else out
    if op == "gated_backward":
        g, u, dh = s["g"].float(), s["u"].float(), s["dh"].float()
        dg, du = dh * u * _act_grad(g, case["act"]), dh * _act(g, case["act"])
        dx = dg @ weight["wg"] + du @ weight["wu"]
        return dx.to(dt), (dg.T @ x).to(dt), (du.T @ x).to(dt)
    g, u = x @ weight["wg"].T, x @ weight["wu"].T
    h = _act(g, case["act"]) * u
    return (h.to(dt), g.to(dt), u.to(dt)) if case["save"] else h.to(dt)


# ------------------------------------------------------- the framework's calls


def _own(s):
    import brovisionml_b200 as bv

    case = s["case"]
    op = case["op"]
    if op == "norm":
        return bv.rms_norm(s["x"], s["w"], s.get("r"), eps=EPS)
    if op == "norm_e4m3":
        return bv.rms_norm_e4m3(s["x"], s["w"], s.get("r"), eps=EPS)
    if op == "norm_backward":
        return bv.rms_norm_backward(s["dy"], s["x"], s["w"], s.get("r"), eps=EPS)
    if op == "linear":
        return bv.linear(s["x"], s["w"], s["b"], act=case["act"], residual=s["r"])
    if op == "linear_e4m3":
        return bv.linear(s["x"], s["w"], s["b"], act=case["act"], residual=s["r"],
                         x_scale=s["xs"], w_scale=s["ws"], out_dtype=TYPES[case["dtype"]])
    if op == "linear_backward":
        out = bv.linear_backward(s["dy"], s["x"], s["w"], s["z"], act=case["act"],
                                 bias=case["bias"])
        return out if case["bias"] else out[:2]
    if op == "gated":
        return bv.gated_linear(s["x"], s["wg"], s["wu"], act=case["act"], save=case["save"])
    if op == "gated_e4m3":
        return bv.gated_linear(s["x"], s["wg"], s["wu"], act=case["act"], save=case["save"],
                               x_scale=s["xs"], gate_scale=s["wgs"], up_scale=s["wus"],
                               out_dtype=TYPES[case["dtype"]])
    return bv.gated_linear_backward(s["dh"], s["x"], s["wg"], s["wu"], s["g"], s["u"],
                                    act=case["act"])


def run(state):
    if own:
        return _own(state)
    return _plain(state)


def work(case):
    op, T, K, N = case["op"], case["T"], case["K"], case.get("N", 0)
    e = 4 if case["dtype"] == "fp32" else 2
    if op.startswith("norm"):
        we = 4 if K % 16 == 0 or case["dtype"] == "fp32" else 2
        res = 1 if case["residual"] else 0
        if op == "norm":
            return {"bytes": T * K * e * (2 + 2 * res) + K * we, "flops": 6 * T * K}
        if op == "norm_e4m3":
            return {"bytes": T * K * (e * (1 + 2 * res) + 1) + 4 * T + K * we, "flops": 8 * T * K}
        return {"bytes": T * K * e * (3 + res) + 2 * K * we, "flops": 14 * T * K}
    i = 1 if op.endswith("e4m3") else 2  # bytes of an input element
    scales = 4 * (T + N) if i == 1 else 0
    if op == "linear_backward":
        z = 1 if case["act"] != "none" else 0
        return {"bytes": 2 * (T * N * (1 + z) + 2 * T * K + 2 * N * K) + 4 * N * case["bias"],
                "flops": 4 * T * N * K}
    if op.startswith("linear"):
        return {"bytes": i * (T + N) * K + scales + 2 * T * N * (1 + case["residual"])
                + 4 * N * case["bias"], "flops": 2 * T * N * K}
    if op == "gated_backward":
        return {"bytes": 2 * (3 * T * N + 2 * T * K + 4 * N * K), "flops": 8 * T * N * K}
    return {"bytes": i * (T + 2 * N) * K + scales + 4 * N * (i == 1)
            + 2 * T * N * (3 if case["save"] else 1), "flops": 4 * T * N * K}


# ------------------------------------------------------------- in 64 bits

_SQRT2PI = math.sqrt(2 * math.pi)
_EXACT_ACT = {
    "none": (lambda z: z, lambda z: z * 0 + 1),
    "relu": (lambda z: z.clamp_min(0), lambda z: z.sign().clamp_min(0)),
    "sigmoid": (torch.sigmoid, lambda z: torch.sigmoid(z) * torch.sigmoid(-z)),
    "tanh": (torch.tanh, lambda z: torch.cosh(z.clamp(-300, 300)).pow(-2)),
    "silu": (lambda z: z * torch.sigmoid(z),
             lambda z: torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z)),
    "gelu": (lambda z: z * torch.special.ndtr(z),
             lambda z: torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / _SQRT2PI),
}


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    for n in ("x", "w", "wg", "wu"):
        if n + "s" in d:
            d[n] = torch.einsum("ij,i->ij", d[n], d[n + "s"])
    op = case["op"]
    if op in ("norm", "norm_e4m3"):
        t = torch.add(d["x"], d["r"]) if "r" in d else d["x"]
        size = (torch.linalg.vector_norm(t, dim=1) ** 2 / case["K"] + EPS).sqrt()
        y = torch.einsum("ij,i,j->ij", t, 1 / size, d["w"])
        first = [y]
        if op == "norm_e4m3":
            # the 8-bit value itself: nearest on the grid of three fraction bits, ties to even
            scale = torch.linalg.vector_norm(y, ord=float("inf"), dim=1) / E4M3_MAX
            v = y / scale[:, None]
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
            first = [torch.round(v / step) * step, scale]
        first += [t] if "r" in d else []
        return tuple(first) if len(first) > 1 else first[0]
    if op == "norm_backward":
        t, dy = d["x"], d["dy"]
        m = torch.einsum("ij,ij->i", t, t) / case["K"] + EPS
        dot = torch.einsum("ij,ij,j->i", dy, t, d["w"]) / case["K"]
        dx = (torch.einsum("ij,j,i->ij", dy, d["w"], m ** -0.5)
              - torch.einsum("ij,i->ij", t, dot * m ** -1.5))
        if "r" in d:
            dx = dx + d["r"]
        return dx, torch.einsum("ij,ij,i->j", dy, t, m ** -0.5)
    f, df = _EXACT_ACT[case["act"]]
    if op == "linear_backward":
        dz = d["dy"] * df(d["z"]) if "z" in d else d["dy"]
        out = (torch.einsum("tn,nk->tk", dz, d["w"]), torch.einsum("tn,tk->nk", dz, d["x"]))
        return out + (dz.sum(0),) if case["bias"] else out
    if op.startswith("linear"):
        y = f(torch.einsum("tk,nk->tn", d["x"], d["w"]) + d.get("b", 0.0))
        return y + d["r"] if "r" in d else y
    if op == "gated_backward":
        both = torch.cat([d["dh"] * d["u"] * df(d["g"]), d["dh"] * f(d["g"])], 1)
        dx = both @ torch.cat([d["wg"], d["wu"]])
        dw = torch.einsum("tn,tk->nk", both, d["x"])
        return dx, dw[:case["N"]], dw[case["N"]:]
    g = torch.einsum("tk,nk->tn", d["x"], d["wg"])
    u = torch.einsum("tk,nk->tn", d["x"], d["wu"])
    return (f(g) * u, g, u) if case["save"] else f(g) * u
