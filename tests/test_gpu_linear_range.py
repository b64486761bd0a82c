"""The linear layer where its numbers leave a type's range, on the GPU."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_gpu_nn import _normal, nn  # noqa: E402,F401


@pytest.mark.parametrize("rows,inner,outer", [(40, 45, 40), (70000, 45, 40), (70000, 300, 40), (3000, 20, 300)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_sums_beyond_float16(nn, act, rows, inner, outer):
    """x W^T of 90000 and -90000: the result is that or 0, in float32, and a'(z) is 1
    or 0, so that the gradients are those of a product without activation whose dy
    is masked.  Every product and sum of those is exact: dy is 2^-8 of an integer."""
    g = torch.Generator().manual_seed(5)
    x = torch.zeros(rows, inner, dtype=torch.float16)
    w = _normal(1, outer, inner, dtype=torch.float16)
    x[:, 0] = 300.0
    w[:, 0] = 300.0 * (1.0 - 2.0 * (torch.arange(outer, device="cuda") % 3 == 0))
    dy = (torch.randint(-1, 2, (rows, outer), generator=g) * 2.0 ** -8).cuda()
    x = x.cuda()
    y, z = nn.linear_forward(x, w, None, None, act, torch.float32, keep=True)
    live = (w[:, 0] > 0).expand(rows, outer)
    assert torch.equal(y, torch.where(live, 90000.0, 0.0))
    assert torch.equal(z, torch.where(live, 65504.0, -65504.0).half())
    w = torch.where(torch.arange(inner, device="cuda") == 0, w, 0.0)
    got, want = nn.linear_backward(dy, x, w, z, act), nn.linear_backward(dy * live, x, w)
    assert all(torch.isfinite(t).all() and torch.equal(t, v) for t, v in zip(got, want))
    for checkpoint in (None, "mx8"):
        b = torch.zeros(outer, dtype=torch.float16, device="cuda", requires_grad=True)
        xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
        nn.linear(xs, ws, b, None, act, torch.float32, checkpoint).backward(dy)
        assert torch.equal(b.grad, want[2]) and torch.isfinite(xs.grad).all() and torch.isfinite(ws.grad).all()


def test_a_nan_stays_one(nn):
    x = torch.ones(40, 45, dtype=torch.float16, device="cuda")
    x[3, 2] = float("nan")
    y, z = nn.linear_forward(x, torch.ones(40, 45, dtype=torch.float16, device="cuda"), activation="silu", keep=True)
    assert torch.isnan(z[3]).all() and torch.isnan(y[3]).all() and torch.isfinite(z[:3]).all()
