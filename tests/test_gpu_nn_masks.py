"""Dropout's masks from an offset in device memory, and in replays of a graph."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_gpu_nn import DTYPES, IDS, _ffn_operands, _normal, nn  # noqa: E402, F401


def _at(v):
    return torch.tensor([v], dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("offset", [0, 7, 0x1122334455667788, -1])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_offset_tensor_is_the_number(nn, dtype, offset):  # noqa: F811
    x, r = _normal(1, 70, 45, dtype=dtype), _normal(2, 70, 45, dtype=dtype)
    assert torch.equal(nn.dropout_add_forward(x, r, 0.3, 5, _at(offset)), nn.dropout_add_forward(x, r, 0.3, 5, offset))
    assert torch.equal(nn.dropout_add_backward(x, 0.3, 5, _at(offset)), nn.dropout_add_backward(x, 0.3, 5, offset))


def test_autograd_with_an_offset_tensor(nn):  # noqa: F811
    x, r = _normal(1, 70, 45).requires_grad_(), _normal(2, 70, 45).requires_grad_()
    dy, at = _normal(3, 70, 45), _at(9)
    got = torch.autograd.grad(nn.dropout_add(x, r, 0.3, 5, at), (x, r), dy)
    want = torch.autograd.grad(nn.dropout_add(x, r, 0.3, 5, 9), (x, r), dy)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    y = nn.dropout_add(x, r, 0.3, 5, at)
    at.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(y, (x, r), dy)


def test_replays_of_a_training_step_drop_other_elements(nn):  # noqa: F811
    x, wg, wu, wd = _ffn_operands(500, 64, 128, torch.bfloat16)
    dy, at = _normal(4, 500, 64, dtype=torch.bfloat16), _at(0)

    def step(offset):
        f = nn.gated_ffn_forward(x, wg, wu, wd)
        y = nn.dropout_add_forward(f, x, 0.25, 3, offset)
        return [y, *nn.gated_ffn_backward(nn.dropout_add_backward(dy, 0.25, 3, offset), x, wg, wu, wd)]

    step(at)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(at)
        at.add_(1)
    at.zero_()
    before = None
    for k in range(5):
        x.copy_(_normal(80 + k // 2, 500, 64, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        eager = step(k)
        assert all(torch.equal(p, q) for p, q in zip(out, eager)), k
        assert before is None or not torch.equal(before, out[0])
        before = out[0].clone()
    assert int(at) == 5


def test_refused_offsets(nn):  # noqa: F811
    x = _normal(1, 8, 16)
    for bad in (torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"),
                torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="offset"):
            nn.dropout_add_forward(x, None, 0.5, 1, bad)


@pytest.mark.parametrize("kind", [np.int32, np.uint32, np.int64, np.uint64])
def test_numpy_seeds(nn, kind):  # noqa: F811
    x = _normal(1, 70, 45)
    assert torch.equal(nn.dropout_add_forward(x, None, 0.3, kind(5), kind(9)), nn.dropout_add_forward(x, None, 0.3, 5, 9))
    with pytest.raises(TypeError):
        nn.dropout_add_forward(x, None, 0.3, 5.0, 9)
