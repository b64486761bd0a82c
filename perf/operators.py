"""The operators of a learned head, as their speed is measured.

A head over the features of a scene's gaussians, or over the pixels of a
rendered view, is a stack of residual blocks x + dropout(ffn(norm(x))): few
features, very many rows.  Its three operators run forward and backward here:

  layer norm           y = (x - mean) rstd weight + bias
  gated feed-forward   y = (a(x Wg^T) * (x Wu^T)) Wd^T,  a = SiLU or GELU
  dropout + residual   y = residual + keep * x / (1 - p)

``run`` calls the library where ``own`` is true and else computes the same in
elementary 32-bit torch operations; ``exact`` computes it in 64 bits.  Row
counts are the gaussian and pixel counts of the benchmark scenes, the width 45
is that of a gaussian's higher spherical harmonics, the others are generic.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5
FRAME = 1297 * 840   # pixels of a view at dataset resolution

# GELU in its tanh form is v * sigmoid(GELU_A v + GELU_B v^3)
GELU_A = 2.0 * math.sqrt(2.0 / math.pi)
GELU_B = 0.044715 * GELU_A

# Philox 4x32 (Salmon, Moraes, Dror and Shaw, SC 2011), seven rounds
PHILOX_M = (0xD2511F53, 0xCD9E8D57)
PHILOX_W = (0x9E3779B9, 0xBB67AE85)
PHILOX_ROUNDS = 7
U32 = 0xFFFFFFFF


def listed():
    return [
        # Some gaussians under an editor's brush, their SH rows normalised: the latency of one call.
        dict(name="norm_small", kind="norm", dtype="f32", rows=257, dim=45),
        # Every pixel's features of one view at dataset resolution.
        dict(name="norm_frame", kind="norm", dtype="bf16", rows=FRAME, dim=64),
        # A training step over the gaussians of a mid-sized scene.
        dict(name="norm_grad_scene", kind="norm_grad", dtype="bf16", rows=500_000, dim=128),
        # The same over a point-cloud-sized scene's SH rows: an odd width, rows off the 16-byte grid.
        dict(name="norm_grad_odd", kind="norm_grad", dtype="f32", rows=120_000, dim=45),
        # A batch of probe points through a wide block: few rows, latency.
        dict(name="ffn_small", kind="ffn", dtype="bf16", rows=256, dim=128, hidden=512, act="silu"),
        # Inference over one view: the ordinary width and expansion.
        dict(name="ffn_frame", kind="ffn", dtype="bf16", rows=FRAME, dim=64, hidden=256, act="silu"),
        # Full precision over a point-cloud-sized scene.
        dict(name="ffn_f32", kind="ffn", dtype="f32", rows=120_000, dim=48, hidden=192, act="gelu"),
        # A training step of a unit-sized scene in full precision.
        dict(name="ffn_grad_small", kind="ffn_grad", dtype="f32", rows=10_000, dim=32, hidden=128, act="silu"),
        # A training step over the gaussians of a mid-sized scene.
        dict(name="ffn_grad_scene", kind="ffn_grad", dtype="bf16", rows=500_000, dim=64, hidden=256, act="silu"),
        # A wide block at sizes that fit no tile.
        dict(name="ffn_grad_wide", kind="ffn_grad", dtype="f16", rows=65_543, dim=200, hidden=1000, act="gelu"),
        # Regularised training on a whole view.
        dict(name="drop_frame", kind="drop", dtype="f16", rows=FRAME, dim=64, p=0.1),
        # Its backward over SH rows.
        dict(name="drop_grad_odd", kind="drop_grad", dtype="f32", rows=120_000, dim=45, p=0.25),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "ffn", "ffn", "ffn_grad", "ffn_grad", "drop", "drop_grad"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    case = dict(kind=kind, dtype=dtype)
    if kind in ("ffn", "ffn_grad"):
        case["dim"] = _log_int(rng, 12, 256)
        case["hidden"] = _log_int(rng, 24, 1100)
        # within the work of ffn_frame and ffn_grad_wide
        most = (FRAME * 64 * 256 if kind == "ffn" else 65_543 * 200 * 1000) // (case["dim"] * case["hidden"])
        if dtype == "f32":
            most //= 8
        case["rows"] = _log_int(rng, 20, max(40, min(most, FRAME if kind == "ffn" else 500_000)))
        case["act"] = rng.choice(["silu", "gelu"])
        return case
    case["dim"] = _log_int(rng, 7, 1500)
    most = {"norm": FRAME * 64, "norm_grad": 500_000 * 128, "drop": FRAME * 64, "drop_grad": FRAME * 32}[kind]
    if dtype == "f32":
        most //= 2
    case["rows"] = _log_int(rng, 20, max(40, min(most // case["dim"], FRAME)))
    if kind in ("drop", "drop_grad"):
        case["p"] = rng.choice([0.05, 0.1, 0.25, 0.5])
    return case


def _inputs(case, seed):
    """The named float32 inputs of a case before they take its type."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    rows, dim, kind = case["rows"], case["dim"], case["kind"]
    if kind in ("norm", "norm_grad"):
        # rows of different brightness and contrast
        t = dict(x=normal(rows, dim) * (0.5 + normal(rows, 1).abs()) + 0.5 * normal(rows, 1),
                 weight=1.0 + 0.1 * normal(dim))
        if kind == "norm":
            t["bias"] = 0.1 * normal(dim)
        else:
            t["dy"] = 0.05 * normal(rows, dim)
        return t
    if kind in ("ffn", "ffn_grad"):
        hidden = case["hidden"]
        t = dict(x=normal(rows, dim), w_gate=normal(hidden, dim) / math.sqrt(dim),
                 w_up=normal(hidden, dim) / math.sqrt(dim), w_down=normal(dim, hidden) / math.sqrt(hidden))
        if kind == "ffn_grad":
            t["dy"] = 0.05 * normal(rows, dim)
        return t
    if kind == "drop":
        return dict(x=normal(rows, dim), residual=normal(rows, dim))
    return dict(dy=0.05 * normal(rows, dim))


def prepare(case, seed):
    state = {k: v.to(DTYPES[case["dtype"]]) for k, v in _inputs(case, seed).items()}
    state["kind"] = case["kind"]
    if case["kind"] == "norm_grad":   # what the forward pass left
        x = state["x"].float()
        state["mean"] = x.mean(1)
        state["rstd"] = torch.rsqrt((x - state["mean"][:, None]).square().mean(1) + EPS)
    if "act" in case:
        state["act"] = case["act"]
    if "p" in case:
        state["p"] = case["p"]
        state["seed"] = (seed * 0x9E3779B97F4A7C15 + 0x6D73706C) & 0xFFFFFFFFFFFFFFFF
        state["offset"] = seed & U32   # a training program's step
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from msplat_amd import nn
    kind = s["kind"]
    if kind == "norm":
        return nn.layer_norm_forward(s["x"], s["weight"], s["bias"], EPS)
    if kind == "norm_grad":
        return nn.layer_norm_backward(s["dy"], s["x"], s["weight"], s["mean"], s["rstd"])
    if kind == "ffn":
        return nn.gated_ffn_forward(s["x"], s["w_gate"], s["w_up"], s["w_down"], s["act"])
    if kind == "ffn_grad":
        return nn.gated_ffn_backward(s["dy"], s["x"], s["w_gate"], s["w_up"], s["w_down"], s["act"])
    if kind == "drop":
        return nn.dropout_add_forward(s["x"], s["residual"], s["p"], s["seed"], s["offset"])
    return nn.dropout_add_backward(s["dy"], s["p"], s["seed"], s["offset"])


def _keep(rows, dim, p, seed, offset):
    """The dropout mask: Philox words in int64, whose wrapped products hold the unsigned 64-bit ones."""
    blocks = (dim + 3) // 4
    c0 = torch.arange(blocks, device="cuda", dtype=torch.int64).expand(rows, blocks)
    c1 = torch.arange(rows, device="cuda", dtype=torch.int64)[:, None].expand(rows, blocks)
    c2 = torch.full((rows, blocks), offset & U32, device="cuda", dtype=torch.int64)
    c3 = torch.full((rows, blocks), offset >> 32, device="cuda", dtype=torch.int64)
    k0, k1 = seed & U32, seed >> 32
    for _ in range(PHILOX_ROUNDS):
        a, b = c0 * PHILOX_M[0], c2 * PHILOX_M[1]
        c0, c1, c2, c3 = ((b >> 32) & U32) ^ c1 ^ k0, b & U32, ((a >> 32) & U32) ^ c3 ^ k1, a & U32
        k0, k1 = (k0 + PHILOX_W[0]) & U32, (k1 + PHILOX_W[1]) & U32
    words = torch.stack((c0, c1, c2, c3), 2).reshape(rows, 4 * blocks)[:, :dim]
    return words >= int(p * 4294967296.0)


def _gate(g, act):
    """sigmoid of the activation's argument and that argument's derivative: a(g) = g * sigmoid."""
    if act == "silu":
        return torch.sigmoid(g), 1.0
    return torch.sigmoid(g * (GELU_A + GELU_B * g * g)), GELU_A + 3.0 * GELU_B * g * g


def _run_plain(s):
    kind = s["kind"]
    dtype = s["dy" if "dy" in s else "x"].dtype
    if kind == "norm":
        x = s["x"].float()
        mean = x.mean(1)
        d = x - mean[:, None]
        rstd = 1.0 / torch.sqrt((d * d).mean(1) + EPS)
        y = d * rstd[:, None] * s["weight"].float() + s["bias"].float()
        return y.to(dtype), mean, rstd
    if kind == "norm_grad":
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        n = (s["x"].float() - s["mean"][:, None]) * rstd
        dn = dy * s["weight"].float()
        dx = rstd * (dn - dn.mean(1, keepdim=True) - n * (dn * n).mean(1, keepdim=True))
        return dx.to(dtype), (dy * n).sum(0).to(dtype), dy.sum(0).to(dtype)
    if kind == "ffn":
        x = s["x"].float()
        g, u = x @ s["w_gate"].float().t(), x @ s["w_up"].float().t()
        return (((g * _gate(g, s["act"])[0]) * u) @ s["w_down"].float().t()).to(dtype)
    if kind == "ffn_grad":
        x, dy = s["x"].float(), s["dy"].float()
        wg, wu, wd = s["w_gate"].float(), s["w_up"].float(), s["w_down"].float()
        g, u = x @ wg.t(), x @ wu.t()
        sig, slope = _gate(g, s["act"])
        a = g * sig
        dh = dy @ wd
        du = dh * a
        dg = dh * u * (sig + a * (1.0 - sig) * slope)
        dx = dg @ wg + du @ wu
        return dx.to(dtype), (dg.t() @ x).to(dtype), (du.t() @ x).to(dtype), (dy.t() @ (a * u)).to(dtype)
    t = s["x" if kind == "drop" else "dy"].float()
    keep = _keep(t.shape[0], t.shape[1], s["p"], s["seed"], s["offset"])
    t = torch.where(keep, t * (1.0 / (1.0 - s["p"])), 0.0)
    return (s["residual"].float() + t if kind == "drop" else t).to(dtype)


def work(case):
    rows, dim = case["rows"], case["dim"]
    size = 4 if case["dtype"] == "f32" else 2
    n = rows * dim
    kind = case["kind"]
    if kind == "norm":
        return {"bytes": 2 * n * size + 2 * dim * size + 8 * rows, "flops": 8 * n}
    if kind == "norm_grad":
        return {"bytes": 3 * n * size + 3 * dim * size + 8 * rows, "flops": 14 * n}
    if kind == "ffn":
        w = dim * case["hidden"]
        return {"bytes": (2 * n + 3 * w) * size, "flops": 6 * rows * w}
    if kind == "ffn_grad":
        w = dim * case["hidden"]
        return {"bytes": (3 * n + 6 * w) * size, "flops": 16 * rows * w}
    return {"bytes": (3 if kind == "drop" else 2) * n * size, "flops": (2 if kind == "drop" else 1) * n}


def _words64(rows, dim, seed, offset):
    """The Philox words in numpy's unsigned arithmetic, row block by row block."""
    out = np.empty((rows, dim), np.uint32)
    cols = np.arange((dim + 3) // 4, dtype=np.uint64)
    mask, half = np.uint64(U32), np.uint64(32)
    for lo in range(0, rows, 65536):
        hi = min(rows, lo + 65536)
        c = [np.broadcast_to(cols, (hi - lo, len(cols))),
             np.broadcast_to(np.arange(lo, hi, dtype=np.uint64)[:, None], (hi - lo, len(cols))),
             np.full((hi - lo, len(cols)), offset % 2 ** 32, np.uint64),
             np.full((hi - lo, len(cols)), offset // 2 ** 32, np.uint64)]
        key = [seed % 2 ** 32, seed // 2 ** 32]
        for _ in range(PHILOX_ROUNDS):
            first, second = c[0] * np.uint64(PHILOX_M[0]), c[2] * np.uint64(PHILOX_M[1])
            c = [(second >> half) ^ c[1] ^ np.uint64(key[0]), second & mask,
                 (first >> half) ^ c[3] ^ np.uint64(key[1]), first & mask]
            key = [(k + w) % 2 ** 32 for k, w in zip(key, PHILOX_W)]
        out[lo:hi] = np.stack(c, 2).reshape(hi - lo, -1)[:, :dim]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() for k, v in s.items() if torch.is_tensor(v)}
    kind = case["kind"]
    if kind == "norm":
        var, mean = torch.var_mean(d["x"], dim=1, correction=0)
        rstd = (var + EPS) ** -0.5
        y = torch.addcmul(d["bias"], (d["x"] - mean.unsqueeze(1)) * rstd.unsqueeze(1), d["weight"])
        return y, mean, rstd
    if kind == "norm_grad":
        n = (d["x"] - d["mean"].unsqueeze(1)) * d["rstd"].unsqueeze(1)
        dn = d["dy"] * d["weight"]
        c1 = dn.sum(1) / case["dim"]
        c2 = (dn * n).sum(1) / case["dim"]
        dx = (dn - c1.unsqueeze(1) - n * c2.unsqueeze(1)) * d["rstd"].unsqueeze(1)
        return dx, (d["dy"] * n).sum(0), d["dy"].sum(0)
    if kind in ("ffn", "ffn_grad"):
        return _exact_ffn(d, case["act"], kind == "ffn_grad")
    t = d["x" if kind == "drop" else "dy"] / (1.0 - case["p"])
    words = torch.from_numpy(_words64(case["rows"], case["dim"], s["seed"], s["offset"]).astype(np.int64)).cuda()
    t[words < math.floor(case["p"] * 2.0 ** 32)] = 0.0
    return t + d["residual"] if kind == "drop" else t


def _exact_ffn(d, act, grad):
    wg, wu, wd = d["w_gate"], d["w_up"], d["w_down"]
    rows = d["x"].shape[0]
    out = torch.empty_like(d["x"])
    sums = [torch.zeros_like(w) for w in (wg, wu, wd)]
    for lo in range(0, rows, 131072):
        x = d["x"][lo:lo + 131072]
        g, u = torch.mm(x, wg.T), torch.mm(x, wu.T)
        if act == "silu":
            a = g / (1.0 + torch.exp(-g))
            slope = (1.0 + torch.exp(-g) * (1.0 + g)) / (1.0 + torch.exp(-g)) ** 2
        else:
            t = torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3))
            a = 0.5 * g * (1.0 + t)
            slope = 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * math.sqrt(2.0 / math.pi) * (1.0 + 0.134145 * g ** 2)
        if not grad:
            out[lo:lo + 131072] = torch.mm(a * u, wd.T)
            continue
        dy = d["dy"][lo:lo + 131072]
        dh = torch.mm(dy, wd)
        dg, du = dh * u * slope, dh * a
        out[lo:lo + 131072] = torch.mm(dg, wg) + torch.mm(du, wu)
        for total, left, right in zip(sums, (dg, du, dy), (x, x, a * u)):
            total += torch.mm(left.T, right)
    return (out, *sums) if grad else out
