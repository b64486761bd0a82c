"""The linear layer's sums over rows on the GPU: exactly, in integers, and in the mean
square, where the elementwise bounds of many rows' worst case are wide."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import linear_exact as exact  # noqa: E402
import more_oracle as orc  # noqa: E402
from linear_sizes import FEW, ONE_PASS, RESIDENT, SIZES, STREAMED, STREAMED_DX  # noqa: E402
from nn_oracle import U, UT, activation  # noqa: E402
from test_gpu_linear import ACTS, _operands  # noqa: E402
from test_gpu_nn import DTYPES, IDS, _normal, nn  # noqa: E402,F401

SEED = 90


@pytest.mark.parametrize("mx", [False, True], ids=["plain", "mx8"])
@pytest.mark.parametrize("rows,inner,outer", SIZES + FEW + ONE_PASS + RESIDENT + STREAMED + STREAMED_DX)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gradients_exactly(nn, dtype, rows, inner, outer, mx):
    x, w, dy, z = (t.cuda() for t in exact.operands(rows, inner, outer, SEED))
    xk, wk, zk = x.to(dtype), w.to(dtype), z.to(dtype)
    if mx:
        xk, zk = nn.mx8_pack(xk), nn.mx8_pack(zk)
    for i, act in enumerate(ACTS):
        want = [exact.rounded(t, dtype) for t in exact.gradients(x, w, dy, z, act)]
        for dy_dtype in {dtype, DTYPES[(DTYPES.index(dtype) + 1 + i % 2) % 3]}:
            got = nn.linear_backward(dy.to(dy_dtype), xk, wk, zk if act else None, act)
            for g, v, what in zip(got, want, ("dx", "dweight", "dbias")):
                assert g.dtype is dtype and torch.equal(g, v), f"{what} {act} {dy_dtype}"


@pytest.mark.parametrize("rows,inner,outer", ONE_PASS[2:] + RESIDENT + STREAMED[4:9])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gradients_in_the_mean_square(nn, dtype, rows, inner, outer):
    """The roundings of different rows are independent, so that the error of a sum is a
    random walk: its expected square is at most the sum of the squares of each term's
    own error (dz rounded to the type by uT of itself at most, and before that by its
    evaluation's bound) and of U of the partial sum at each of at most `rows` additions,
    and of the result's rounding.  Uniform errors have a third of that; over all
    elements twice the root is far beyond chance."""
    x, w, _ = _operands(rows, inner, outer, dtype)
    z, uT = _normal(51, rows, outer, dtype=dtype, scale=2.0), UT[dtype][0]
    for dy_dtype in {dtype, torch.float32}:
        dy = _normal(50, rows, outer, dtype=dy_dtype)
        got = nn.linear_backward(dy, x, w, z, "silu")
        (_, dw, db), _ = orc.linear_grad(dy, x, w, z, "silu", dtype)
        a, da, q = activation(z.double(), "silu")
        dz = dy.double() * da
        e_s = (8 + 4 * q) * U   # as in linear_grad
        e_dz = dy.double().abs() * ((e_s + 6 * U) * (1.0 + a.abs() * (1.0 + q)) + e_s * a.abs() * (1.0 + q)) + 2 * U * dz.abs()
        walk = rows * U ** 2 * dz.square() + e_dz.square()
        allowed = (walk + (uT * dz).square() + UT[dtype][1] ** 2).t() @ x.double().square(), walk.sum(0)
        for g, v, e, what in zip(got[1:], (dw, db), allowed, ("dweight", "dbias")):
            error = float((g.double() - v).square().sum()) ** 0.5
            bound = 2 * float((e + (uT * v).square() + UT[dtype][1] ** 2).sum()) ** 0.5
            assert error <= bound, f"{what} {dy_dtype}: {error:.3g} where {bound:.3g} is allowed"
