"""The mean-square checks of the learned-head operators without a GPU: that their
sizes reach every kernel, and that they fail for a sum that misses rows."""
from __future__ import annotations

import os

import pytest
import torch

import nn_dispatch
import nn_norms as norms
from msplat_amd import _abi
from nn_sizes import FFN_ALL, FFN_MANY, NORM_MANY

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _operands(rows, dim, hidden, dtype):
    g = torch.Generator().manual_seed(rows + dim)
    shapes = ((rows, dim, 1.0), (rows, dim, 1.0), (hidden, dim, dim ** -0.5), (hidden, dim, dim ** -0.5),
              (dim, hidden, hidden ** -0.5))
    return [(s * torch.randn(a, b, generator=g)).to(dtype) for a, b, s in shapes]


# ranges of the operator's sizes in which its launch rules change
ROWS = (1, 40, 300, 4096, 4100, 8200, 9000, 16384, 16400, 17000, 32768, 33000, 65543, 70000, 131079, 140000, 262149)
HIDDEN = (1, 3, 7, 8, 24, 64, 200, 256, 400, 800, 1100, 1800, 5000)


@pytest.mark.parametrize("size", [4, 2])
def test_sizes_reach_every_kernel(size):
    reach = set()
    for dim in list(range(1, 40)) + list(range(40, 257, 3)) + [128, 192, 256]:
        for hidden in HIDDEN:
            for rows in ROWS:
                plan = nn_dispatch.Plan(size, rows, dim, hidden)
                reach.update(plan.forward() + plan.backward())
    tested = set()
    for sizes in FFN_ALL:
        plan = nn_dispatch.Plan(size, *sizes)
        tested.update(plan.forward() + plan.backward())
    assert not reach - tested, sorted(reach - tested, key=str)
    shapes = {(p.lanes, p.pieces) for p in (nn_dispatch.NormPlan(size, 1, d) for d in range(1, 8193))}
    assert shapes == {(p.lanes, p.pieces) for p in (nn_dispatch.NormPlan(size, *s) for s in NORM_MANY)}


def test_launch_rules_are_the_librarys():
    """Through the workspaces' sizes, which follow from them."""
    if not os.path.exists(_abi.LIB_PATH):
        pytest.skip("libmsplat_hip.so not built")
    lib = _abi.load()
    for dtype, number in DTYPES.items():
        size = torch.empty(0, dtype=dtype).element_size()
        for dim in (1, 3, 5, 8, 17, 33, 45, 64, 65, 100, 128, 150, 180, 192, 200, 256):
            for hidden in HIDDEN:
                for rows in (0,) + ROWS:
                    plan = nn_dispatch.Plan(size, rows, dim, hidden)
                    assert lib.msplat_hip_gated_ffn_workspace(rows, dim, hidden, number) == plan.forward_workspace()
                    assert lib.msplat_hip_gated_ffn_backward_workspace(rows, dim, hidden, number) == \
                        plan.backward_workspace(), (dtype, rows, dim, hidden)
        for rows, dim in NORM_MANY + [(1, 1), (1000, 45)]:
            assert lib.msplat_hip_layer_norm_backward_workspace(rows, dim, number) == \
                nn_dispatch.NormPlan(size, rows, dim).backward_workspace(dim)


@pytest.mark.parametrize("rows,dim,hidden", [s for s in FFN_MANY if s[0] * s[2] < 8_000_000])
def test_a_lost_block_of_rows_fails(rows, dim, hidden):
    """In bf16, whose limits are the widest, for one block of 32 rows (the last,
    short one where it has 16 rows or more, else the one before), and for one
    of the rows at edges."""
    dtype = torch.bfloat16
    ops = _operands(rows, dim, hidden, dtype)
    plan = nn_dispatch.Plan(2, rows, dim, hidden)
    whole = norms.gated_ffn(*ops, "silu")
    last = rows // 32 * 32 if rows % 32 >= 16 else (rows // 32 - 1) * 32
    block = slice(last, min(last + 32, rows))
    part = norms.gated_ffn(ops[0][block], ops[1][block], *ops[2:], "silu")
    for (v, q2, n), (lost, _, _), what in list(zip(whole, part, norms.NAMES))[2:]:
        norms.near(v.to(dtype), v, q2, n, dim, what)
        with pytest.raises(AssertionError, match="error"):
            norms.near((v - lost).to(dtype), v, q2, n, dim, what)
    edges = plan.edge_rows()
    assert edges[0] == 0 and edges[-1] == rows - 1
    dy, x = ops[0][edges], ops[1][edges]
    whole = norms.gated_ffn(dy, x, *ops[2:], "silu")
    part = norms.gated_ffn(dy[-1:], x[-1:], *ops[2:], "silu")
    for (v, q2, n), (lost, _, _), what in list(zip(whole, part, norms.NAMES))[2:]:
        with pytest.raises(AssertionError, match="error"):
            norms.near((v - lost).to(dtype), v, q2, n, dim, what)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_a_lost_row_of_five_fails(dtype):
    terms = torch.randn(5, 1000, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    norms.columns_near(terms.sum(0).to(dtype), terms, "whole")
    with pytest.raises(AssertionError, match="error"):
        norms.columns_near(terms[:4].sum(0).to(dtype), terms, "four of five")
