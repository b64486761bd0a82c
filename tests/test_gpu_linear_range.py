"""The linear layer where its numbers leave a type's range, on the GPU."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import more_oracle as more  # noqa: E402
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


# few rows' kernels; one pass; parts of dW and dx by rows in LDS; dx from a streamed contraction
@pytest.mark.parametrize("rows,inner,outer", [(40, 45, 40), (700, 64, 250), (3000, 300, 150), (20000, 300, 300)])
@pytest.mark.parametrize("own_dz", [False, True])
def test_an_infinite_gradient_stays_where_it_is(nn, own_dz, rows, inner, outer):
    """In its row of dx, its output's row of dweight and its element of dbias, of a width that
    no piece divides."""
    x, w = _normal(2, rows, inner, dtype=torch.bfloat16), _normal(3, outer, inner, dtype=torch.bfloat16)
    dy = _normal(4, rows, outer, dtype=torch.float32 if own_dz else torch.bfloat16)
    z = _normal(5, rows, outer, dtype=torch.bfloat16)
    for act in (None, "silu"):
        clean = nn.linear_backward(dy, x, w, z, act)
        far = dy.clone()
        far[7, outer - 1], far[8, 1] = float("inf"), float("nan")
        dx, dw, db = nn.linear_backward(far, x, w, z, act)
        rest = torch.ones(rows, dtype=torch.bool, device="cuda")
        rest[7:9] = False
        assert torch.equal(dx[rest], clean[0][rest]) and not torch.isfinite(dx[7]).any() and torch.isnan(dx[8]).all()
        rest = torch.ones(outer, dtype=torch.bool, device="cuda")
        rest[outer - 1] = rest[1] = False
        assert torch.equal(dw[rest], clean[1][rest]) and torch.equal(db[rest], clean[2][rest])
        for t in (dw, db):
            assert not torch.isfinite(t[outer - 1]).any() and torch.isnan(t[1]).all()


def test_far_offsets_of_streamed_weights(nn):
    """Rows beyond 2^32 elements of x, the residual, dy and z, where the weights are streamed,
    and packed rows beyond 2^32 bytes."""
    rows, inner, outer = 132000, 300, 3
    stride = (1 << 15) + 8
    assert rows * stride > 1 << 32

    def far(t):
        out = torch.empty(rows * stride, dtype=t.dtype, device="cuda").as_strided(t.shape, (stride, 1))
        return out.copy_(t)

    x, w = _normal(6, rows, inner, dtype=torch.bfloat16), _normal(7, outer, inner, dtype=torch.bfloat16)
    r, dy = _normal(8, rows, outer, dtype=torch.bfloat16), _normal(9, rows, outer, dtype=torch.bfloat16)
    want = nn.linear_forward(x, w, None, r, "silu", keep=True)
    grads = nn.linear_backward(dy, x, w, want[1], "silu")
    xs, rs = far(x), far(r)
    got = nn.linear_forward(xs, w, None, rs, "silu", keep=True)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    del rs
    dys, zs = far(dy), far(want[1])
    assert all(torch.equal(p, q) for p, q in zip(nn.linear_backward(dys, xs, w, zs, "silu"), grads))
    wide = nn.linear_backward(dy.float(), x, w, want[1], "silu")
    assert all(torch.equal(p, q) for p, q in zip(nn.linear_backward(dys.float(), xs, w, zs, "silu"), wide))
    del xs, dys, zs
    rows = (1 << 32) // 288 + 77
    x = torch.zeros(rows, 288, dtype=torch.bfloat16, device="cuda")
    x[-40:] = _normal(10, 40, 288, dtype=torch.bfloat16)
    w, b = nn.mx8_pack(_normal(11, outer, 288, dtype=torch.bfloat16)), _normal(12, outer)
    m = nn.mx8_pack(x)
    del x
    y = nn.linear_forward(m, w, b, out_dtype=torch.float32)
    assert torch.equal(y[:-40], b.expand(rows - 40, outer))
    xv, wv = (nn.mx8_unpack(t, torch.float32) for t in (nn.Mx8(m.data[-40:], m.scales[-40:], 288, m.dtype), w))
    value, _, bound, _ = more.linear(xv, wv, b, None, None, torch.float32)
    more.near(y[-40:], value, bound, "the last rows")
