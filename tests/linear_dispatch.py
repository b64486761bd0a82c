"""Which kernels of the linear layer a call runs, by its sizes: the launch rules of
csrc/linear.hpp restated, so that the tests can show that their sizes reach every
kernel.  The sizes of the workspaces, which the library works out by the same rules
without a GPU, hold this file to them.  size: bytes of an element of x and weight
(2 also for products of 8 bits)."""
from __future__ import annotations

CUS = 256
LDS_BYTES = 160 * 1024


def ceil_div(a, b):
    return -(-a // b)


def product(size, rows, inner, outer):
    """The kernels of a product [rows, inner] x [outer, inner]^T, and its workspace."""
    kbs, blocks = ceil_div(inner, 64 // size), ceil_div(outer, 32)
    if ceil_div(rows, 64) * blocks <= (1024 if inner > 512 else 2048):
        return {("few", 1 if rows <= 16 else 4)}, 0
    if kbs <= 8:
        kbs += kbs in (5, 7)
        slices = ceil_div(blocks, LDS_BYTES // (kbs * 2048 + 128))
        return {("all", kbs), ("all in slices", slices > 1)}, 0
    slices = ceil_div(blocks, 8)
    nb, steps = ceil_div(blocks, slices), ceil_div(kbs, 2)
    turn = 256 * max(CUS // slices, 1)
    tail = rows > turn and 0 < rows % turn <= 1024
    return {("stream", nb), ("tail", tail), ("odd steps", steps % 2 == 1)}, slices * steps * 2 * 2 * nb * 1024


def up(n, m=16):
    return ceil_div(n, m) * m


def backward(size, rows, inner, outer, activation, same_type):
    """The kernels of a backward call for all gradients, and its workspace."""
    own = not same_type
    wide, deep = (256, 64) if size == 4 else (256, 128)
    one = not own and (outer <= wide and inner <= deep or outer <= deep and inner <= wide)
    if inner <= 64:
        n, k = 256, 64
    elif outer <= 64:
        n, k = 64, 256
    elif size == 4:
        n, k = 256, 64
    else:
        n, k = (256, 128) if inner <= 128 or outer > 128 else (128, 256)
    tiles = ceil_div(outer, n) * ceil_div(inner, k)
    groups = min(ceil_div(rows, 128 // size), max(CUS // tiles, 1))
    kernels = {("one pass" if one else "parts", n, k), ("fold", groups > 32)}
    work = up(groups * (outer * inner + outer) * 4)
    if own:
        tx = 1
        while tx < 256 and tx * 8 < outer:
            tx *= 2
        work += up(ceil_div(rows, max(ceil_div(rows, 1024), 1024 // tx)) * outer * 4)
        kernels.add("dz")
    if own or not one and activation:
        work += up(rows * outer * size)
    if not one:
        dx, more = product(size, rows, outer, inner)
        kernels |= {("dx", *k) for k in dx}
        work += more
    return kernels, work
