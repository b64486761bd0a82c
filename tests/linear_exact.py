"""A linear layer's gradients in which every rounding is exact, so that a test may ask
for equality: small integers, and an activation's arguments so far out that its
derivative is 1 or 0.  A lost, doubled or misplaced step of rows, a partial sum
added to another place or sums of fewer bits than 24 show."""
from __future__ import annotations

import torch


def operands(rows, inner, outer, seed):
    """x, w, dy of integers in [-2, 2] and z of 128 and -128 (also in 8 bits), on the CPU."""
    g = torch.Generator().manual_seed(seed)
    x, w, dy = (torch.randint(-2, 3, s, generator=g).float() for s in ((rows, inner), (outer, inner), (rows, outer)))
    z = 256.0 * torch.randint(0, 2, (rows, outer), generator=g) - 128.0
    return x, w, dy, z


def gradients(x, w, dy, z, act):
    """dx, dweight, dbias in 64 bits.  Every sum of magnitudes is below 2^24, so that 32-bit
    sums are exact in any order; the results are then rounded once."""
    x, w, dz = x.double(), w.double(), (dy if act is None else dy * (z > 0)).double()
    assert 4 * max(x.shape[0], w.shape[0]) < 1 << 24
    return dz @ w, dz.t() @ x, dz.sum(0)


def rounded(t, dtype):
    return t.float().to(dtype)
