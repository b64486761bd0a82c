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
from nn_sizes import FFN_ALL, FFN_MANY  # noqa: E402
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
