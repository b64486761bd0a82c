"""8-bit rows, the root-mean-square norm and the linear layer in 64 bits, from
their formulas, with elementwise bounds on the rounding of the 32-bit evaluation
(nn_oracle has the conventions)."""
from __future__ import annotations

import torch

from nn_oracle import U, UT, activation

LARGEST = {torch.float32: 1.875 * 2.0 ** 127, torch.bfloat16: 1.875 * 2.0 ** 127, torch.float16: 61440.0}


def blocks(x):
    """[rows, dim] as [rows, blocks, 32], zeros behind dim."""
    rows, dim = x.shape
    n = -(-dim // 32)
    return torch.nn.functional.pad(x, (0, 32 * n - dim)).view(rows, n, 32)


def exponents(amax):
    """The least e in [-126, 127] with amax <= 448 2^e."""
    e = torch.full(amax.shape, -126.0, dtype=torch.float64)
    for _ in range(260):
        e += (amax > 448.0 * torch.exp2(e)) & (e < 127)
    return e


def e4m3(v):
    """|v| <= 448 at the nearest e4m3 number, ties to the even one; NaN stays."""
    e = (torch.frexp(v.abs().nan_to_num(0.0)).exponent - 1).clamp(min=-6).double()
    step = torch.exp2(e - 3.0)
    return torch.round(v / step) * step


def mx8(x):
    """(values [rows, dim], codes [rows, blocks]) of x packed, exactly."""
    rows, dim = x.shape
    v = x.double().cpu()
    v = torch.where(torch.isfinite(v), v.clamp(-LARGEST[x.dtype], LARGEST[x.dtype]), float("nan"))
    b = blocks(v)
    e = exponents(b.abs().nan_to_num(0.0).amax(2))
    s = torch.exp2(e)[:, :, None]
    return (e4m3(b / s) * s).view(rows, -1)[:, :dim], (e + 127).to(torch.int64)


def mx8_bound(y, e_y):
    """How far a packed number may be from y where what was packed is off by e_y:
    half a step of 2^-4 of it, or of 2^-10 of the scale, which may be the next one
    where the block's largest is on the border."""
    rows, dim = y.shape
    size = y.abs() + e_y
    s = torch.exp2(exponents(blocks(size).amax(2)))
    low = (2.0 ** -10 * s)[:, :, None].expand(-1, -1, 32).reshape(rows, -1)[:, :dim]
    return e_y + torch.maximum(2.0 ** -4 * size, low)


def rms_norm(total, weight, eps):
    """y, rstd and their bounds from the rounded sum.  No sum of a row is deeper
    than 40 additions (layer_norm in nn_oracle); 1 / sqrt takes two roundings."""
    uT, tiny = UT[total.dtype]
    t, w = total.double().cpu(), weight.double().cpu()
    ms = t.square().mean(1)
    rstd = (ms + eps).rsqrt()
    e_rstd = rstd * (0.5 * 44 * U + 4 * U)
    y = t * rstd[:, None] * w
    e_32 = (t.abs() * e_rstd[:, None]) * w.abs() + 3 * U * y.abs()
    return y, rstd, e_32, e_32 + (uT + U) * y.abs() + tiny, e_rstd


def rms_norm_grad(dy, total, weight, rstd, dtotal):
    """dx, dweight and their bounds, total's values given in 64 bits."""
    uT, tiny = UT[dy.dtype]
    rows = dy.shape[0]
    dy, t, w, rstd = (v.double().cpu() for v in (dy, total, weight, rstd))
    r = rstd[:, None]
    n, g = t * r, dy * w
    c = (g * n).mean(1, keepdim=True)
    dt = torch.zeros_like(dy) if dtotal is None else dtotal.double().cpu()
    dx = r * (g - n * c) + dt
    e_c = 46 * U * (g * n).abs().mean(1, keepdim=True)
    e_dx = r * (n.abs() * e_c + 5 * U * (g.abs() + (n * c).abs())) + U * dt.abs() + (uT + U) * dx.abs() + tiny
    dw = (dy * n).sum(0)
    e_dw = (rows + 4) * U * (dy * n).abs().sum(0) + uT * dw.abs() + tiny
    return (dx, dw), (e_dx, e_dw)


def linear(x, w, bias, residual, act, out_dtype):
    """y, z = x w^T + bias and their bounds, z in x's type and before it was rounded.
    x and w as their values (64 bits or less); a product's sum over dim terms is
    off by dim U of their magnitudes at most.  The kernels start the sum from the
    bias: every partial sum is then at most |b| + sum |x| |w| in magnitude, so that
    each of the dim additions rounds by U of that at most, dim U (|b| + sum |x| |w|) in all."""
    uT, tiny = UT[out_dtype]
    x, w = x.double(), w.double()
    dim = x.shape[1]
    z = x @ w.t()
    e_z = dim * U * (x.abs() @ w.abs().t())
    if bias is not None:
        z = z + bias.double()
        e_z = e_z + dim * U * bias.double().abs() + U * z.abs()
    if act is None:
        y, e_y = z, e_z
    else:
        y, _, q = activation(z, act)
        e_y = 1.2 * e_z + y.abs() * (8 + 4 * q) * U
    if residual is not None:
        y = y + residual.double()
        e_y = e_y + U * y.abs()
    return y, z, e_y + (uT + U) * y.abs() + tiny, e_z


def linear_grad(dy, x, w, z, act, dtype):
    """(dx, dweight, dbias) and their bounds; x and z as their values.  In 16-bit
    types dz is rounded to the type for the products, not for dbias."""
    uT, tiny = UT[dtype]
    dy, x, w = (t.double() for t in (dy, x, w))
    rows, outer = dy.shape
    dz, e_dz = dy, torch.zeros_like(dy)
    if act is not None:
        z = z.double()
        a, da, q = activation(z, act)
        e_s = (8 + 4 * q) * U
        dz = dy * da
        # a' = s + a (1 - s) q' with the errors of a and s, z q' < 1 + 3 q
        e_dz = dy.abs() * ((e_s + 6 * U) * (1.0 + a.abs() * (1.0 + q)) + e_s * a.abs() * (1.0 + q)) + 2 * U * dz.abs()
    e_t = e_dz + (uT + U) * dz.abs() + tiny
    dx = dz @ w
    e_dx = e_t @ w.abs() + outer * U * (dz.abs() @ w.abs()) + (uT + U) * dx.abs() + tiny
    dw = dz.t() @ x
    e_dw = e_t.t() @ x.abs() + rows * U * (dz.abs().t() @ x.abs()) + (uT + U) * dw.abs() + tiny
    db = dz.sum(0)
    e_db = e_dz.sum(0) + rows * U * dz.abs().sum(0) + (uT + U) * db.abs() + tiny
    return (dx, dw, db), (e_dx, e_dw, e_db)


def near(got, want, bound, what):
    """nn_oracle.within on the tensors' own device."""
    got = got.double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} vs {tuple(want.shape)}"
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = (got - want).abs() - bound
    assert (over <= 0).all(), (f"{what}: {int((over > 0).sum())} of {got.numel()} beyond the bound, worst by "
                               f"{float(over.max()):.3g} where that is {float(bound.flatten()[over.argmax()]):.3g}")
