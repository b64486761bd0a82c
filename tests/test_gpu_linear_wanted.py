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


@pytest.mark.parametrize("rows,inner,outer,y_dtype", [(700, 300, 300, 2), (700, 64, 256, 2), (5000, 300, 300, 0)])
def test_dbias_by_itself_writes_its_own_sums_alone(nn, rows, inner, outer, y_dtype):
    """Neither the weight's sums nor dy in its type go to the workspace: at most a row of
    sums of each of the pass's 256 workgroups, or of the 1024 that make dy's."""
    import ctypes
    from msplat_amd import _abi
    lib = _abi.load()
    _, w, _ = _operands(rows, inner, outer, torch.bfloat16)
    dy = _normal(50, rows, outer, dtype=[torch.float32, None, torch.bfloat16][y_dtype])
    want = nn.linear_backward(dy, None, w, wanted=(False, False, True))[2]
    size = lib.msplat_hip_linear_backward_workspace(rows, inner, outer, 2, y_dtype, 2)
    ws = torch.full((size,), 0xAB, dtype=torch.uint8, device="cuda")
    got = torch.empty(outer, dtype=torch.bfloat16, device="cuda")
    a = _abi.LinearGradArgs(None, rows, inner, outer, 2, y_dtype, 2, dy.data_ptr(), outer, None, 0, None, w.data_ptr(), inner,
                            None, 0, None, None, 0, None, got.data_ptr(), ws.data_ptr(), ws.nbytes)
    torch.cuda.synchronize()
    _abi.check(lib.msplat_hip_linear_backward(ctypes.byref(a)))
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    steps = (rows + 63) // 64 if y_dtype == 2 else rows // 4   # workgroups at most
    assert int((ws != 0xAB).sum()) <= min(steps, 1024) * outer * 4 < size / 8
