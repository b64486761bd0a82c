"""Gradients of the linear layer that do not take its input, on the GPU."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_gpu_linear import ACTS, _operands  # noqa: E402
from test_gpu_nn import DTYPES, IDS, _normal, nn  # noqa: E402,F401

# few rows; one pass; parts of dW; an input narrower than a piece; dx as a streamed product
SIZES = [(3, 45, 40), (700, 64, 256), (700, 300, 300), (500, 3, 2), (66000, 60, 300)]


@pytest.mark.parametrize("rows,inner,outer", SIZES)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_without_x(nn, dtype, rows, inner, outer):
    x, w, _ = _operands(rows, inner, outer, dtype)
    for i, act in enumerate(ACTS):
        z = _normal(51, rows, outer, dtype=dtype, scale=2.0) if act else None
        for out_dtype in {dtype, DTYPES[(DTYPES.index(dtype) + i) % 3]}:
            dy = _normal(50, rows, outer, dtype=out_dtype)
            dx, _, db = nn.linear_backward(dy, x, w, z, act)
            for wanted in ((True, False, True), (True, False, False), (False, False, True)):
                got = nn.linear_backward(dy, None, w, z, act, wanted)
                assert [t is not None for t in got] == list(wanted)
                assert got[0] is None or torch.equal(got[0], dx)
                assert got[2] is None or torch.equal(got[2], db)
