"""The linear layer on the GPU at the sizes that reach the kernels which test_gpu_linear's
lists leave out."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import more_oracle as orc  # noqa: E402
from linear_sizes import STREAMED_DX, THREE_BLOCKS  # noqa: E402
from test_gpu_linear import ACTS, _check_backward, _check_forward, _operands  # noqa: E402
from test_gpu_nn import DTYPES, IDS, _normal, nn  # noqa: E402,F401


@pytest.mark.parametrize("rows,inner,outer", THREE_BLOCKS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_forward(nn, dtype, rows, inner, outer):
    x, w, b = _operands(rows, inner, outer, dtype)
    for act in ACTS:
        for out_dtype in DTYPES:
            r = _normal(40, rows, outer, dtype=out_dtype)
            y, z = nn.linear_forward(x, w, b, r, act, out_dtype, keep=True)
            _check_forward(y, x, w, b, r, act, out_dtype, f"y {act} in {out_dtype}")
            _, want, _, e_z = orc.linear(x, w, b, None, None, dtype)
            uT, tiny = orc.UT[dtype]
            orc.near(z, want, e_z + (uT + orc.U) * want.abs() + tiny, "z")
            assert torch.equal(nn.linear_forward(x, w, b, r, act, out_dtype), y)
    _check_forward(nn.linear_forward(x, w), x, w, None, None, None, dtype, "product alone")


@pytest.mark.parametrize("rows,inner,outer", STREAMED_DX)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_backward(nn, dtype, rows, inner, outer):
    for act, out_dtype in ((None, dtype), ("silu", dtype), ("gelu", DTYPES[(DTYPES.index(dtype) + 1) % 3])):
        _check_backward(nn, dtype, rows, inner, outer, act, False, out_dtype)
