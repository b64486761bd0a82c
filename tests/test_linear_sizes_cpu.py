"""The sizes of the linear layer's tests reach every kernel, by the launch rules restated
in linear_dispatch.  No GPU."""
from __future__ import annotations

import pytest

import linear_dispatch as rules
from linear_sizes import FEW, ONE_PASS, RESIDENT, SIZES, STREAMED, STREAMED_DX, THREE_BLOCKS
from test_nn_cpu import BF16, F16, F32, lib  # noqa: F401

FORWARD = SIZES + FEW + RESIDENT + STREAMED
PRODUCTS = {("few", 1), ("few", 4), *(("all", n) for n in (1, 2, 3, 4, 6, 8)), ("all in slices", False),
            ("all in slices", True), *(("stream", n) for n in range(1, 9)), ("tail", False), ("tail", True),
            ("odd steps", False), ("odd steps", True)}


def test_the_rules_are_the_librarys(lib):  # noqa: F811
    for size, dtype in ((4, F32), (2, F16), (2, BF16)):
        other = F16 if dtype == F32 else F32
        for rows, inner, outer in FORWARD + ONE_PASS + THREE_BLOCKS + [(1 << 20, 1000, 1000), (900, 5000, 777), (0, 40, 9)]:
            assert lib.msplat_hip_linear_workspace(rows, inner, outer, dtype) == rules.product(size, rows, inner, outer)[1]
            for act in (0, 1, 2):
                for y in (dtype, other):
                    got = lib.msplat_hip_linear_backward_workspace(rows, inner, outer, dtype, y, act)
                    assert got == rules.backward(size, rows, inner, outer, act != 2, y == dtype)[1], (rows, inner, outer, dtype, y, act)


@pytest.mark.parametrize("size", [4, 2])
def test_every_forward_kernel_is_reached(size):
    reached = set().union(*(rules.product(size, *s)[0] for s in FORWARD + THREE_BLOCKS))
    assert reached == PRODUCTS


@pytest.mark.parametrize("size", [4, 2])
def test_every_backward_kernel_is_reached(size):
    reached = set()
    for rows, inner, outer in FORWARD + ONE_PASS + STREAMED_DX:
        for act in (False, True):
            for same in (True, False):
                reached |= rules.backward(size, rows, inner, outer, act, same)[0]
    shapes = [(256, 64), (64, 256)] + ([(256, 128), (128, 256)] if size == 2 else [])
    want = {(w, *s) for w in ("one pass", "parts") for s in shapes} | {("fold", False), ("fold", True), "dz"}
    assert reached - {k for k in reached if k[0] == "dx"} == want
    assert PRODUCTS - {k[1:] for k in reached if k[0] == "dx"} == set()
