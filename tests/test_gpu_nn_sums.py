"""Sums over many rows, and every kernel form of the learned-head operators:
errors in the mean square, which a lost block of rows shows in (nn_norms), and
gradients that come from chosen rows alone."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import nn_dispatch  # noqa: E402
import nn_norms as norms  # noqa: E402
import nn_oracle as orc  # noqa: E402
from nn_sizes import FFN_ALL, FFN_MANY, NORM_MANY  # noqa: E402
from test_gpu_nn import DTYPES, IDS, _ffn_operands, _normal, nn  # noqa: E402, F401


@pytest.mark.parametrize("rows,dim,hidden", FFN_ALL)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gated_ffn_in_the_mean_square(nn, dtype, rows, dim, hidden):  # noqa: F811
    for act in ("silu", "gelu"):
        ops = _ffn_operands(rows, dim, hidden, dtype)
        dy = _normal(30, rows, dim, dtype=dtype)
        got = (nn.gated_ffn_forward(*ops, act), *nn.gated_ffn_backward(dy, *ops, act))
        want = norms.gated_ffn(dy, *ops, act)
        for g, (v, q2, n), what in zip(got, want, norms.NAMES):
            norms.near(g, v, q2, n, dim, f"{what} {act}")
        for g, (v, q2, n), what in zip(got[:2], want, norms.NAMES):
            norms.rows_near(g, v, q2, n, dim, f"{what} {act}")
        again = (nn.gated_ffn_forward(*ops, act), *nn.gated_ffn_backward(dy, *ops, act))
        assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("rows,dim,hidden", FFN_MANY)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_weight_gradients_of_rows_at_edges(nn, dtype, rows, dim, hidden):  # noqa: F811
    """dy is zero but in the rows on both sides of the edges of the row groups
    and of the last blocks: every gradient is that of these rows alone."""
    ops = _ffn_operands(rows, dim, hidden, dtype)
    plan = nn_dispatch.Plan(ops[0].element_size(), rows, dim, hidden)
    all_edges = torch.tensor(plan.edge_rows(), device="cuda")
    for edges in (all_edges, all_edges[-3:], all_edges[:1]):
        dy = torch.zeros(rows, dim, dtype=dtype, device="cuda")
        dy[edges] = _normal(31, len(edges), dim, dtype=dtype)
        got = nn.gated_ffn_backward(dy, *ops)
        want = norms.gated_ffn(dy[edges], ops[0][edges], *ops[1:], "silu")
        for g, (v, q2, n), what in zip(got[1:], want[2:], norms.NAMES[2:]):
            norms.near(g, v, q2, n, dim, what)
        norms.rows_near(got[0][edges], *want[1], dim, "dx")
        rest = torch.ones(rows, dtype=torch.bool, device="cuda")
        rest[edges] = False
        assert (got[0][rest] == 0).all()


@pytest.mark.parametrize("rows,dim", NORM_MANY)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_layer_norm_of_many_rows(nn, dtype, rows, dim):  # noqa: F811
    """More rows than workgroups take in one turn: rows as in calls of few rows,
    bit for bit, and the sums over them in the mean square."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (2 * torch.randn(rows, dim, generator=g, device="cuda")).to(dtype)
    dy = torch.randn(rows, dim, generator=g, device="cuda").to(dtype)
    w, b = 1 + _normal(3, dim, dtype=dtype, scale=0.1), _normal(4, dim, dtype=dtype)
    y, mean, rstd = nn.layer_norm_forward(x, w, b)
    dx, dweight, dbias = nn.layer_norm_backward(dy, x, w, mean, rstd)
    plan = nn_dispatch.NormPlan(x.element_size(), rows, dim)
    step = plan.backward_groups * plan.at_once
    assert step < rows and plan.forward_groups * plan.at_once < rows
    for at in range(0, rows, step):
        part = slice(at, at + step)
        few = nn.layer_norm_forward(x[part], w, b)
        assert all(torch.equal(p, q[part]) for p, q in zip(few, (y, mean, rstd))), at
        assert torch.equal(nn.layer_norm_backward(dy[part], x[part], w, mean[part], rstd[part])[0], dx[part]), at
    n = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    norms.columns_near(dweight, dy.double() * n, "dweight")
    norms.columns_near(dbias, dy.double(), "dbias")
    edges = torch.tensor(sorted({0, plan.at_once - 1, step - 1, step, rows - 1}), device="cuda")
    few = torch.zeros_like(dy)
    few[edges] = dy[edges]
    _, dweight, dbias = nn.layer_norm_backward(few, x, w, mean, rstd)
    norms.columns_near(dweight, (dy.double() * n)[edges], "dweight of rows at edges")
    norms.columns_near(dbias, dy.double()[edges], "dbias of rows at edges")
