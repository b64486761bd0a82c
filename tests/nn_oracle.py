"""Learned-head operators in 64 bits, from their formulas, with elementwise
bounds on the rounding of the 32-bit evaluation.

The bounds are first-order worst cases: a sum of n products is off by at most
n u times the sum of their magnitudes (u = 2^-24), a function by its
argument's error times its slope, and a value rounded to its type T by uT of
itself plus half of T's smallest step.
"""
from __future__ import annotations

import math

import numpy as np
import torch

U = 2.0 ** -24
# unit roundoff (2^-p for p significant bits: 24, 11, 8) and half the smallest
# subnormal of each type
UT = {torch.float32: (2.0 ** -24, 0.0), torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 0.0)}


def layer_norm(x, weight, bias, eps):
    """y, mean, rstd and their bounds.  The kernel adds at most 32 elements a
    lane and joins at most 256 lanes: no sum is deeper than 40 additions."""
    uT, tiny = UT[x.dtype]
    x, w, b = (t.double().cpu() for t in (x, weight, bias))
    mean = x.mean(1)
    d = x - mean[:, None]
    var = d.square().mean(1)
    rstd = (var + eps).rsqrt()
    n = d * rstd[:, None]
    y = n * w + b
    e_mean = 42 * U * x.abs().mean(1)
    # d has the mean's error and its own rounding; var is its mean square
    e_d = e_mean[:, None] + U * d.abs()
    e_var = (2 * d.abs() * e_d + e_d.square()).mean(1) + 44 * U * var
    e_rstd = rstd * (0.5 * e_var / (var + eps) + 4 * U)
    e_n = e_d * rstd[:, None] + d.abs() * e_rstd[:, None] + 2 * U * n.abs()
    e_y = (e_n + U * n.abs()) * w.abs() + (uT + U) * y.abs() + U * b.abs() + tiny
    return (y, mean, rstd), (e_y, e_mean, e_rstd)


def layer_norm_grad(dy, x, weight, mean, rstd):
    """dx, dweight, dbias and their bounds, for the given mean and rstd.  The
    columns' sums run over the rows in an order of any depth."""
    uT, tiny = UT[x.dtype]
    rows = x.shape[0]
    dy, x, w, mean, rstd = (t.double().cpu() for t in (dy, x, weight, mean, rstd))
    r = rstd[:, None]
    n = (x - mean[:, None]) * r
    g = dy * w
    c1, c2 = g.mean(1, keepdim=True), (g * n).mean(1, keepdim=True)
    dx = r * (g - c1 - n * c2)
    e_n = 2 * U * n.abs()
    e_c1 = 43 * U * g.abs().mean(1, keepdim=True)
    e_c2 = 46 * U * (g * n).abs().mean(1, keepdim=True)
    parts = g.abs() + c1.abs() + (n * c2).abs()
    e_dx = r.abs() * (e_c1 + n.abs() * e_c2 + e_n * c2.abs() + 5 * U * parts) + (uT + U) * dx.abs() + tiny
    dw, db = (dy * n).sum(0), dy.sum(0)
    e_dw = (rows + 4) * U * (dy * n).abs().sum(0) + uT * dw.abs() + tiny
    e_db = rows * U * dy.abs().sum(0) + uT * db.abs() + tiny
    return (dx, dw, db), (e_dx, e_dw, e_db)


GELU_C = math.sqrt(2.0 / math.pi)


def activation(g, act):
    """a(g), its derivative, and the size of the sigmoid's argument."""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1.0 + g * (1.0 - s)), g.abs()
    z = 2.0 * GELU_C * (g + 0.044715 * g ** 3)
    s = torch.sigmoid(z)
    return g * s, s + g * s * (1.0 - s) * 2.0 * GELU_C * (1.0 + 0.134145 * g ** 2), z.abs()


def gated_ffn(x, wg, wu, wd, act):
    """y in the tensors' own precision (differentiable)."""
    return (activation(x @ wg.t(), act)[0] * (x @ wu.t())) @ wd.t()


def _rounded(v, uT, tiny, f32=U):
    return (uT + f32) * v.abs() + tiny


def _forward(x, wg, wu, act):
    dim = x.shape[1]
    g, u = x @ wg.t(), x @ wu.t()
    e_g, e_u = dim * U * (x.abs() @ wg.abs().t()), dim * U * (x.abs() @ wu.abs().t())
    a, da, z = activation(g, act)
    # |a'| < 1.2; the sigmoid's argument is rounded a few times (relative to
    # its size), the exponential, the quotient and the products once each
    e_s = (8 + 4 * z) * U
    e_a = 1.2 * e_g + a.abs() * e_s
    return g, u, a, da, z, e_g, e_u, e_a, e_s


def gated_ffn_bounds(x, wg, wu, wd, act):
    """y and its bound."""
    uT, tiny = UT[x.dtype]
    x, wg, wu, wd = (t.double().cpu() for t in (x, wg, wu, wd))
    g, u, a, da, z, e_g, e_u, e_a, e_s = _forward(x, wg, wu, act)
    h, y = a * u, (a * u) @ wd.t()
    e_h = e_a * u.abs() + a.abs() * e_u + _rounded(h, uT, tiny)
    e_y = e_h @ wd.abs().t() + h.shape[1] * U * (h.abs() @ wd.abs().t()) + _rounded(y, uT, tiny)
    return y, e_y


def gated_ffn_grad_bounds(dy, x, wg, wu, wd, act):
    """(dx, dw_gate, dw_up, dw_down) and their bounds."""
    uT, tiny = UT[x.dtype]
    dy, x, wg, wu, wd = (t.double().cpu() for t in (dy, x, wg, wu, wd))
    rows, dim = x.shape
    hidden = wg.shape[0]
    g, u, a, da, z, e_g, e_u, e_a, e_s = _forward(x, wg, wu, act)
    dh = dy @ wd
    e_dh = dim * U * (dy.abs() @ wd.abs())
    h, du, dg = a * u, dh * a, dh * u * da
    # |a''| < 1.2; a' = s + a (1 - s) z' with the errors of a and s, z' < 1 + z
    e_da = 1.2 * e_g + (e_s + 6 * U) * (1.0 + a.abs() * (1.0 + z)) + e_s * a.abs() * (1.0 + z)
    e_h = e_a * u.abs() + a.abs() * e_u + _rounded(h, uT, tiny)
    e_du = e_dh * a.abs() + dh.abs() * e_a + _rounded(du, uT, tiny, 2 * U)
    e_dg = e_dh * (u * da).abs() + dh.abs() * (e_u * da.abs() + u.abs() * e_da) + _rounded(dg, uT, tiny, 3 * U)
    dx = dg @ wg + du @ wu
    mag = dg.abs() @ wg.abs() + du.abs() @ wu.abs()
    e_dx = e_dg @ wg.abs() + e_du @ wu.abs() + 2 * hidden * U * mag + _rounded(dx, uT, tiny)
    out, err = [dx], [e_dx]
    for left, e_left, right in ((dg, e_dg, x), (du, e_du, x)):
        v = left.t() @ right
        out.append(v)
        err.append(e_left.t() @ right.abs() + rows * U * (left.abs().t() @ right.abs()) + _rounded(v, uT, tiny))
    v = dy.t() @ h
    out.append(v)
    err.append(dy.abs().t() @ e_h + rows * U * (dy.abs().t() @ h.abs()) + _rounded(v, uT, tiny))
    return out, err


PHILOX_M = (0xD2511F53, 0xCD9E8D57)
PHILOX_W = (0x9E3779B9, 0xBB67AE85)


def philox(counter, key, rounds):
    """Philox 4x32 over arrays of counters: four uint64 arrays holding 32 bits each."""
    c = [np.asarray(v, np.uint64) for v in counter]
    k = [int(v) for v in key]
    mask, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(PHILOX_M[0]), c[2] * np.uint64(PHILOX_M[1])
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & mask, (a >> half) ^ c[3] ^ np.uint64(k[1]), a & mask]
        k = [(v + w) & 0xFFFFFFFF for v, w in zip(k, PHILOX_W)]
    return c


def keep_mask(rows, dim, p, seed, offset):
    blocks = (dim + 3) // 4
    c0, c1 = np.meshgrid(np.arange(blocks), np.arange(rows))
    full = np.zeros((rows, blocks), np.uint64)
    words = philox((c0, c1, full + np.uint64(offset & 0xFFFFFFFF), full + np.uint64(offset >> 32)),
                   (seed & 0xFFFFFFFF, seed >> 32), 7)
    w = np.stack(words, 2).reshape(rows, 4 * blocks)[:, :dim]
    return torch.from_numpy(w.astype(np.int64) >= int(p * 2.0 ** 32))


def dropout_add(x, residual, p, seed, offset):
    """The operator's own 32-bit arithmetic: one product, one sum, one rounding."""
    keep = keep_mask(x.shape[0], x.shape[1], p, seed, offset)
    scale = np.float32(1.0 / (1.0 - p)) if p < 1.0 else np.float32(0.0)
    t = torch.where(keep, x.float().cpu() * torch.tensor(scale), torch.zeros(()))
    return (t if residual is None else residual.float().cpu() + t).to(x.dtype)


def within(got, want, bound, what):
    got = got.double().cpu()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} vs {tuple(want.shape)}"
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - bound
    assert (over <= 0).all(), (f"{what}: {int((over > 0).sum())} of {got.numel()} beyond the bound, worst "
                               f"{float((got - want).abs().max()):.3g}, bound there {float(bound.flatten()[over.argmax()]):.3g}")
