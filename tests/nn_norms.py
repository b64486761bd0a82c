"""The learned-head operators in 64 bits on the tensors' own device, with bounds
on their errors in the mean square.

An elementwise worst case grows with the number of rows that a weight's gradient
sums, the value only with its root, so over many rows a worst case lets a lost
block of rows pass.  In the mean square errors grow as the values do: rounding v
to a type is off by less than uT |v| / sqrt(3), errors of a sum's terms add up
in the square, and its n additions in 32 bits are each off by U of a partial
sum, together below U sqrt(n) of the terms' root sum of squares and the value.
An output v = sum of a_k b_k with a_k rounded to the type then has

    error^2 < uT^2 / 3 (q^2 + v^2),   q^2 = sum of a_k^2 b_k^2

on average over an output's elements; the limits allow uT^2 (q^2 + v^2), sqrt(3)
of it, where there are 1000 elements or more, and twice that where there are
fewer.  The products, activations and their derivatives that come before are off
by sqrt(dim) + 12 roundings in 32 bits.
"""
from __future__ import annotations

import torch

import nn_oracle as orc

NAMES = ("y", "dx", "dw_gate", "dw_up", "dw_down")


def gated_ffn(dy, x, wg, wu, wd, act):
    """(value, q^2, additions of the longest sum) of y, dx, dw_gate, dw_up, dw_down."""
    dy, x, wg, wu, wd = (t.double() for t in (dy, x, wg, wu, wd))
    g, u = x @ wg.t(), x @ wu.t()
    a, da, _ = orc.activation(g, act)
    dh = dy @ wd
    h, du, dg = a * u, dh * a, dh * u * da
    rows, hidden = g.shape
    out = [(h @ wd.t(), h.square() @ wd.square().t(), hidden),
           (dg @ wg + du @ wu, dg.square() @ wg.square() + du.square() @ wu.square(), 2 * hidden)]
    for left, right in ((dg, x), (du, x), (dy, h)):
        out.append((left.t() @ right, left.square().t() @ right.square(), rows))
    return out


def limit(dtype, additions, dim):
    """Of an output's error in the mean square, over that of its terms and value."""
    return orc.UT[dtype][0] + orc.U * (additions ** 0.5 + dim ** 0.5 + 12)


def near(got, value, q2, additions, dim, what):
    """The whole output's error."""
    most = limit(got.dtype, additions, dim) * (1 if value.numel() >= 1000 else 2)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    error, size = float((got.double() - value).norm()), float((q2 + value.square()).sum().sqrt())
    assert error <= most * size, f"{what}: error {error:.3g}, {error / size:.3g} of the size, at most {most:.3g}"


def rows_near(got, value, q2, additions, dim, what):
    """Every row's error: four limits, seven standard deviations of a row of one element."""
    most = 4 * limit(got.dtype, additions, dim)
    over = (got.double() - value).norm(dim=1) - most * (q2 + value.square()).sum(1).sqrt()
    assert float(over.max()) <= 0, f"{what}: {int((over > 0).sum())} rows off, the first {int((over > 0).nonzero()[0])}"


def columns_near(got, terms, what):
    """got = terms.sum(0) of a sum over rows whose terms are exact up to 32-bit
    rounding: only the result is rounded to its type."""
    value, rows = terms.sum(0), terms.shape[0]
    size = float(value.norm())
    walk = orc.U * (rows ** 0.5 + 12) * float((terms.square().sum(0) + value.square()).sum().sqrt())
    most = orc.UT[got.dtype][0] * (1 if value.numel() >= 1000 else 2) * size + walk
    error = float((got.double() - value).norm())
    assert error <= most, f"{what}: error {error:.3g}, at most {most:.3g}, size {size:.3g}"
