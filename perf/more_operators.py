"""More operators of a learned head, as their speed is measured.

Around the blocks that perf/operators.py measures, a head over the pixels of a
view or the features of a scene's gaussians has plain products at its ends, a
norm after each residual addition, and activations that are kept for the
backward pass:

  mx8           rows kept in 8 bits: e4m3 elements, one power of two for each
                32 adjacent columns, packed and restored
  rms           t = x + residual,  y = t rstd weight, in the type or in mx8
  rms_grad      its gradients, t in the type or in mx8
  linear        y = residual + a(x W^T + bias),  a = none, SiLU or GELU
  linear_mx     the same with x and W in mx8
  linear_grad   its gradients, x and z = x W^T + bias in the type or in mx8

``run`` calls the library where ``own`` is true and else computes the same in
elementary 32-bit torch operations; ``exact`` computes it in 64 bits.  Row
counts are the gaussian and pixel counts of the benchmark scenes, the width 45
is that of a gaussian's higher spherical harmonics, the others are generic.
What is held in 8 bits is returned as the values it stands for.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5
FRAME = 1297 * 840   # pixels of a view at dataset resolution

# GELU in its tanh form is v * sigmoid(GELU_A v + GELU_B v^3)
GELU_A = 2.0 * math.sqrt(2.0 / math.pi)
GELU_B = 0.044715 * GELU_A

BLOCK = 32                # columns of a scale
E4M3_MAX = 448.0
LARGEST = {torch.float32: 1.875 * 2.0 ** 127, torch.bfloat16: 1.875 * 2.0 ** 127, torch.float16: 61440.0}


def listed():
    return [
        # Some gaussians under an editor's brush, their SH rows normalised: the latency of one call.
        dict(name="rms_small", kind="rms", dtype="f32", rows=257, dim=45, mx=False),
        # Between two blocks over every pixel of a view: the sum and its norm.
        dict(name="rms_frame", kind="rms", dtype="bf16", rows=FRAME, dim=64, mx=False),
        # The same over the gaussians of a mid-sized scene, for a product that takes 8 bits.
        dict(name="rms_mx_scene", kind="rms", dtype="bf16", rows=500_000, dim=128, mx=True),
        # A training step's backward from a checkpoint in 8 bits.
        dict(name="rms_grad_scene", kind="rms_grad", dtype="bf16", rows=500_000, dim=128, mx=True),
        # Checkpoints of a point-cloud-sized scene's SH rows: an odd width in full precision.
        dict(name="mx8_odd", kind="mx8", dtype="f32", rows=120_000, dim=45),
        # Checkpoints of a view's features.
        dict(name="mx8_frame", kind="mx8", dtype="bf16", rows=FRAME, dim=64),
        # A few probe points: the latency of one call.
        dict(name="linear_small", kind="linear", dtype="bf16", rows=8, inner=256, outer=1000, act="silu", bias=True,
             residual=False),
        # The hidden layer of a plain head over one view.
        dict(name="linear_frame", kind="linear", dtype="bf16", rows=FRAME, inner=64, outer=256, act="gelu", bias=True,
             residual=False),
        # A wide product at sizes that fit no tile, added to the residual.
        dict(name="linear_wide", kind="linear", dtype="f16", rows=65_543, inner=1000, outer=200, act="none", bias=True,
             residual=True),
        # Inference over a scene's gaussians from 8 bits.
        dict(name="linear_mx_scene", kind="linear_mx", dtype="bf16", rows=500_000, inner=256, outer=256, act="silu",
             bias=True, residual=False),
        # A training step over the gaussians of a mid-sized scene.
        dict(name="linear_grad_scene", kind="linear_grad", dtype="bf16", rows=500_000, inner=64, outer=256, act="silu",
             mx=False),
        # Full precision over a point-cloud-sized scene, from checkpoints in 8 bits.
        dict(name="linear_grad_mx", kind="linear_grad", dtype="f32", rows=120_000, inner=48, outer=192, act="gelu",
             mx=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["mx8", "rms", "rms", "rms_grad", "linear", "linear", "linear_mx", "linear_grad", "linear_grad"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    case = dict(kind=kind, dtype=dtype)
    if kind in ("mx8", "rms", "rms_grad"):
        case["dim"] = _log_int(rng, 7, 1500)
        most = (FRAME * 64 if kind == "mx8" else 500_000 * 128) // (2 if dtype == "f32" else 1)
        case["rows"] = _log_int(rng, 20, max(40, min(most // case["dim"], FRAME)))
        if kind != "mx8":
            case["mx"] = rng.choice([False, True])
        return case
    case["inner"], case["outer"] = _log_int(rng, 5, 1100), _log_int(rng, 3, 1100)
    # within the work of linear_wide, linear_mx_scene and linear_grad_scene, and the bytes of the last two
    products = {"linear": 65_543 * 1000 * 200, "linear_mx": 500_000 * 256 * 256, "linear_grad": 500_000 * 64 * 256}[kind]
    if dtype == "f32":
        products //= 4
    most = min(products // (case["inner"] * case["outer"]), 500_000 * 320 // (case["inner"] + case["outer"]) // 2, FRAME)
    case["rows"] = _log_int(rng, 1, max(40, most))
    case["act"] = rng.choice(["none", "silu", "gelu"])
    if kind == "linear_grad":
        case["mx"] = rng.choice([False, True])
    else:
        case["bias"], case["residual"] = rng.choice([False, True]), rng.choice([False, True])
    return case


def _exponents(t):
    """Of each block the least e with amax <= 448 2^e, amax over its finite elements."""
    amax = torch.where(torch.isfinite(t), t.abs(), 0.0).amax(-1)
    mantissa, e = torch.frexp(amax)   # amax = mantissa 2^e, mantissa in [0.5, 1)
    e = e - 9 + (mantissa > 0.875)
    return torch.where(amax > 0, e, -126).clamp(-126, 127)


def _pack(t, dtype):
    """(data [rows, blocks * 32] in e4m3, scales [rows, 4 * ceil(columns / 128)] as bytes e + 127) of a float32
    matrix, whose numbers beyond the type's largest that 8 bits hold count as that one."""
    rows, dim = t.shape
    blocks = -(-dim // BLOCK)
    t = torch.where(torch.isfinite(t), t.clamp(-LARGEST[dtype], LARGEST[dtype]), math.nan)
    t = torch.nn.functional.pad(t, (0, blocks * BLOCK - dim)).view(rows, blocks, BLOCK)
    e = _exponents(t)
    data = torch.ldexp(torch.ldexp(t, -(e // 2)[..., None]), (e // 2 - e)[..., None]).to(torch.float8_e4m3fn)
    scales = torch.zeros(rows, 4 * -(-dim // 128), dtype=torch.uint8, device=t.device)
    scales[:, :blocks] = (e + 127).to(torch.uint8)
    return data.view(rows, blocks * BLOCK), scales


def _unpack(packed, dim):
    """The float32 values of packed rows."""
    data, scales = packed
    rows, blocks = data.shape[0], data.shape[1] // BLOCK
    e = scales[:, :blocks].int()[..., None] - 127
    t = data.float().view(rows, blocks, BLOCK)
    return torch.ldexp(torch.ldexp(t, e // 2), e - e // 2).view(rows, blocks * BLOCK)[:, :dim]


def _inputs(case, seed):
    """The named float32 inputs of a case before they take its type."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    rows, kind = case["rows"], case["kind"]
    if kind in ("mx8", "rms", "rms_grad"):
        dim = case["dim"]
        # rows of different brightness and contrast
        t = dict(x=normal(rows, dim) * (0.5 + normal(rows, 1).abs()) + 0.5 * normal(rows, 1))
        if kind != "mx8":
            t["weight"] = 1.0 + 0.1 * normal(dim)
        if kind == "rms":
            t["residual"] = normal(rows, dim)
        if kind == "rms_grad":
            t["dy"], t["dtotal"] = 0.05 * normal(rows, dim), 0.05 * normal(rows, dim)
        return t
    inner, outer = case["inner"], case["outer"]
    t = dict(x=normal(rows, inner), weight=normal(outer, inner) / math.sqrt(inner))
    if kind == "linear_grad":
        t["dy"] = 0.05 * normal(rows, outer)
        if case["act"] != "none":
            t["z"] = normal(rows, outer)
        return t
    if case["bias"]:
        t["bias"] = 0.1 * normal(outer)
    if case["residual"]:
        t["residual"] = normal(rows, outer)
    return t


def prepare(case, seed):
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    state = {k: v.to(dtype) for k, v in _inputs(case, seed).items()}
    if kind == "rms_grad":   # what the forward pass left
        state["rstd"] = torch.rsqrt(state["x"].float().square().mean(1) + EPS)
    # what is kept in 8 bits: a checkpoint, the features that a norm wrote, weights
    packed = {"linear_mx": ("x", "weight"), "linear_grad": ("x", "z"), "rms_grad": ("x",)}.get(kind, ())
    if kind == "linear_mx" or case.get("mx"):
        for k in packed:
            if k in state:
                state[k] = _pack(state[k].float(), dtype)
    if kind == "linear_mx" and "bias" in state:
        state["bias"] = state["bias"].float()
    state.update(kind=kind, dtype=dtype, mx=case.get("mx", False), act=case.get("act", "none"),
                 inner=case.get("inner", case.get("dim")), outer=case.get("outer"))
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from msplat_amd import nn
    kind, act = s["kind"], None if s["act"] == "none" else s["act"]

    def kept(t, dim):
        return nn.Mx8(*t, dim, s["dtype"]) if isinstance(t, tuple) else t

    if kind == "mx8":
        return nn.mx8_unpack(nn.mx8_pack(s["x"]))
    if kind == "rms":
        y, total, rstd = nn.rms_norm_forward(s["x"], s["weight"], s["residual"], EPS, mx8=s["mx"])
        return nn.mx8_unpack(y, torch.bfloat16) if s["mx"] else y, total, rstd
    if kind == "rms_grad":
        return nn.rms_norm_backward(s["dy"], kept(s["x"], s["inner"]), s["weight"], s["rstd"], s["dtotal"])
    if kind == "linear":
        return nn.linear_forward(s["x"], s["weight"], s.get("bias"), s.get("residual"), act)
    if kind == "linear_mx":
        return nn.linear_forward(kept(s["x"], s["inner"]), kept(s["weight"], s["inner"]), s.get("bias"),
                                 s.get("residual"), act)
    z = kept(s["z"], s["outer"]) if act else None
    return nn.linear_backward(s["dy"], kept(s["x"], s["inner"]), s["weight"], z, act)


def _act(v, act):
    if act == "none":
        return v
    return v * torch.sigmoid(v if act == "silu" else v * (GELU_A + GELU_B * v * v))


def _slope(v, act):
    """a'(v) from a(v) = v sigmoid(q(v))."""
    if act == "silu":
        q, dq = v, 1.0
    else:
        q, dq = v * (GELU_A + GELU_B * v * v), GELU_A + 3.0 * GELU_B * v * v
    sig = torch.sigmoid(q)
    return sig + v * sig * (1.0 - sig) * dq


def _run_plain(s):
    kind, dtype = s["kind"], s["dtype"]

    def values(t, dim):
        return _unpack(t, dim) if isinstance(t, tuple) else t.float()

    if kind == "mx8":
        return _unpack(_pack(s["x"].float(), dtype), s["inner"]).to(dtype)
    if kind == "rms":
        total = (s["x"].float() + s["residual"].float()).to(dtype)
        t = total.float()
        rstd = 1.0 / torch.sqrt((t * t).mean(1) + EPS)
        y = t * rstd[:, None] * s["weight"].float()
        return _unpack(_pack(y, dtype), s["inner"]).bfloat16() if s["mx"] else y.to(dtype), total, rstd
    if kind == "rms_grad":
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        n = values(s["x"], s["inner"]) * rstd
        g = dy * s["weight"].float()
        dx = rstd * (g - n * (g * n).mean(1, keepdim=True)) + s["dtotal"].float()
        return dx.to(dtype), (dy * n).sum(0).to(dtype)
    if kind in ("linear", "linear_mx"):
        y = values(s["x"], s["inner"]) @ values(s["weight"], s["inner"]).t()
        if "bias" in s:
            y = y + s["bias"].float()
        y = _act(y, s["act"])
        if "residual" in s:
            y = y + s["residual"].float()
        return y.to(dtype)
    dz = s["dy"].float()
    if s["act"] != "none":
        dz = dz * _slope(values(s["z"], s["outer"]), s["act"])
    x, w = values(s["x"], s["inner"]), s["weight"].float()
    return (dz @ w).to(dtype), (dz.t() @ x).to(dtype), dz.sum(0).to(dtype)


def work(case):
    rows, kind = case["rows"], case["kind"]
    size = 4 if case["dtype"] == "f32" else 2
    packed = 1.0 + 1.0 / BLOCK
    kept = packed if case.get("mx") else size
    if kind in ("mx8", "rms", "rms_grad"):
        dim = case["dim"]
        n = rows * dim
        if kind == "mx8":
            return {"bytes": int(2 * n * (size + packed)), "flops": 2 * n}
        if kind == "rms":
            # 8 bits are written, and read again where their values are returned
            y = 2 * packed + 2 if case["mx"] else size
            return {"bytes": int(n * (3 * size + y)) + dim * size + 4 * rows, "flops": 5 * n}
        return {"bytes": int(n * (3 * size + kept)) + 2 * dim * size + 4 * rows, "flops": 10 * n}
    x, y, w = rows * case["inner"], rows * case["outer"], case["inner"] * case["outer"]
    if kind == "linear_grad":
        z = kept if case["act"] != "none" else 0
        return {"bytes": int(x * (kept + size) + y * (size + z)) + (2 * w + case["outer"]) * size,
                "flops": 4 * rows * w}
    taken = packed if kind == "linear_mx" else size
    return {"bytes": int((x + w) * taken) + y * size * (2 if case["residual"] else 1)
            + (case["outer"] * (4 if kind == "linear_mx" else size) if case["bias"] else 0), "flops": 2 * rows * w}


def _e4m3(v):
    """|v| <= 448 in 64 bits at the nearest e4m3 number, ties to the even one: 3 bits after the point, from 2^-6 down
    steps of 2^-9."""
    step = torch.exp2((torch.frexp(v.abs()).exponent - 1).clamp(min=-6).double() - 3.0)
    return torch.round(v / step) * step


def _exact_kept(v, dtype):
    """What packing makes of a matrix, in 64 bits (finite values)."""
    rows, dim = v.shape
    v = v.clamp(-LARGEST[dtype], LARGEST[dtype])
    out = torch.empty_like(v)
    for lo in range(0, dim, BLOCK):
        part = v[:, lo:lo + BLOCK]
        amax = part.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(torch.clamp(amax, min=2.0 ** -1000) / E4M3_MAX))
        e = torch.where(amax <= E4M3_MAX * torch.exp2(e - 1), e - 1, e)   # where the logarithm fell on the wrong side
        e = torch.where(amax > E4M3_MAX * torch.exp2(e), e + 1, e).clamp(-126, 127)
        out[:, lo:lo + BLOCK] = _e4m3(part * torch.exp2(-e)) * torch.exp2(e)
    return out


def _exact_values(packed, dim):
    data, scales = packed
    e = torch.repeat_interleave(scales.double() - 127.0, BLOCK, 1)[:, :dim]
    return data[:, :dim].double() * torch.exp2(e)


def exact(case, seed):
    s = prepare(case, seed)
    kind, dtype = case["kind"], s["dtype"]

    def values(t, dim):
        return _exact_values(t, dim) if isinstance(t, tuple) else t.double()

    if kind == "mx8":
        return _exact_kept(s["x"].double(), dtype)
    if kind == "rms":
        total = s["x"].double() + s["residual"].double()
        t = total.to(dtype).double()   # the norm is that of the sum as it is kept
        rstd = (t.square().mean(1) + EPS) ** -0.5
        y = t * rstd.unsqueeze(1) * s["weight"].double()
        return _exact_kept(y, dtype) if case["mx"] else y, total, rstd
    if kind == "rms_grad":
        n = values(s["x"], case["dim"]) * s["rstd"].double().unsqueeze(1)
        g = s["dy"].double() * s["weight"].double()
        along = (g * n).sum(1) / case["dim"]
        dx = (g - n * along.unsqueeze(1)) * s["rstd"].double().unsqueeze(1) + s["dtotal"].double()
        return dx, (s["dy"].double() * n).sum(0)
    rows, inner, outer, act = case["rows"], case["inner"], case["outer"], case["act"]
    w = values(s["weight"], inner)
    if kind in ("linear", "linear_mx"):
        out = torch.empty(rows, outer, dtype=torch.float64, device="cuda")
        for lo in range(0, rows, 131072):
            x = tuple(t[lo:lo + 131072] for t in s["x"]) if isinstance(s["x"], tuple) else s["x"][lo:lo + 131072]
            z = torch.mm(values(x, inner), w.T)
            if "bias" in s:
                z += s["bias"].double()
            if act == "silu":
                z = z / (1.0 + torch.exp(-z))
            elif act == "gelu":
                z = 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)))
            out[lo:lo + 131072] = z
        return out + s["residual"].double() if "residual" in s else out
    x, dz = values(s["x"], inner), s["dy"].double()
    if act != "none":
        z = values(s["z"], outer)
        if act == "silu":
            dz = dz * (1.0 + torch.exp(-z) * (1.0 + z)) / (1.0 + torch.exp(-z)) ** 2
        else:
            t = torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
            dz = dz * (0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * math.sqrt(2.0 / math.pi) * (1.0 + 0.134145 * z ** 2))
    return torch.mm(dz, w), torch.mm(dz.T, x), dz.sum(0)
