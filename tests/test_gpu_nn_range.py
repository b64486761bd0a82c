"""Learned-head operators at the ends of their types' ranges and of their sizes."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import nn_norms as norms  # noqa: E402
import nn_oracle as orc  # noqa: E402
from test_gpu_nn import _normal, nn  # noqa: E402, F401


@pytest.mark.parametrize("power", [5, 10, 43, 44, 63, 65, 100, 126])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [2, 20000])
def test_gradients_of_large_gates(nn, rows, dtype, act, power):  # noqa: F811
    """Gates of +-2^power with u = 1, where a is the gate or 0 and a' 1 or 0 (SiLU
    at +-32 within 2^-40: below every type's rounding).  All values are powers of
    two or a sum of two rounded once."""
    gate = 2.0 ** power
    x = torch.ones(rows, 1, dtype=dtype, device="cuda")
    x[1::2] = -1

    def weight(v):
        return torch.full((1, 1), v, dtype=dtype, device="cuda")

    dy = torch.zeros_like(x)
    dy[0], dy[rows - 1] = 1, 1           # a row of each sign
    y = nn.gated_ffn_forward(x, weight(gate), weight(1.0), weight(1.0), act)
    dx, dg, du, dd = nn.gated_ffn_backward(dy, x, weight(gate), weight(1.0), weight(1.0), act)
    # x = 1: g = gate, u = 1, y = gate, dg = u, du = a = gate;  x = -1: all 0 (silu(-32) is 4e-13)
    close = dict(rtol=0, atol=1e-11)
    assert torch.allclose(y[:2].double().flatten().cpu(), torch.tensor([gate, 0.0], dtype=torch.float64), **close)
    want = torch.tensor([gate + gate]).to(dtype)
    assert torch.allclose(dx[0].double().cpu(), want.double(), **close)
    assert torch.allclose(dx[rows - 1].double().cpu(), torch.zeros(1, dtype=torch.float64), rtol=0, atol=1e-9)
    for got, value in ((dg, 1.0), (du, gate), (dd, gate)):
        assert abs(float(got) - value) <= 1e-11 * value, (float(got), value)


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 2 ** 31 - 256), (torch.float16, 2 ** 31 - 2041),
                                       (torch.float32, 2 ** 31 - 1021)], ids=["bf16", "f16", "f32"])
def test_dropout_of_one_row_of_the_largest_width(nn, dtype, dim):  # noqa: F811
    """The step past the row's end does not fit a signed 32-bit index."""
    p, seed, offset = 0.25, 0xFEDCBA9876543210, 0x1122334455667788
    y = nn.dropout_add_forward(torch.ones(dim, dtype=dtype, device="cuda"), None, p, seed, offset)
    kept = torch.tensor(1.0 / (1.0 - p)).to(dtype).cuda()
    count = 0
    for part in y.split(1 << 28):
        zero = part == 0
        assert bool((zero | (part == kept)).all())
        count += part.numel() - int(zero.sum())
    # five standard deviations of the kept share
    assert abs(count / dim - (1 - p)) < 5 * (p * (1 - p) / dim) ** 0.5
    for first in (0, 2 ** 30 - 512, (dim - 1024) // 4 * 4):
        n = min(1024, dim - first)
        columns = np.arange(first // 4, (first + n + 3) // 4)
        words = orc.philox((columns, 0 * columns, 0 * columns + (offset & 0xFFFFFFFF), 0 * columns + (offset >> 32)),
                           (seed & 0xFFFFFFFF, seed >> 32), 7)
        keep = np.stack(words, 1).reshape(-1)[:n] >= np.uint64(int(p * 2.0 ** 32))
        assert torch.equal(y[first:first + n].cpu() != 0, torch.from_numpy(keep)), first


def test_gated_ffn_of_more_rows_than_a_launch_has_threads_for(nn):  # noqa: F811
    """2^30 rows through streamed weights: four threads a row are 2^32."""
    rows, hidden, dtype = 2 ** 30 + 33, 1800, torch.float16
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, 1, generator=g, device="cuda", dtype=dtype)
    ops = [_normal(2 + i, *s, dtype=dtype, scale=f) for i, (s, f) in
           enumerate((((hidden, 1), 1.0), ((hidden, 1), 1.0), ((1, hidden), hidden ** -0.5)))]
    at = torch.tensor([0, 1, 2 ** 29 - 1, 2 ** 29, 2 ** 30 - 1, 2 ** 30, rows - 1], device="cuda")
    dy = torch.zeros_like(x)
    dy[at] = _normal(5, len(at), 1, dtype=dtype)
    want = norms.gated_ffn(dy[at], x[at], *ops, "silu")
    norms.rows_near(nn.gated_ffn_forward(x, *ops)[at], *want[0], 1, "y")
    dx, *grads = nn.gated_ffn_backward(dy, x, *ops)
    norms.rows_near(dx[at], *want[1], 1, "dx")
    for got, (v, q2, n), what in zip(grads, want[2:], norms.NAMES[2:]):
        norms.near(got, v, q2, n, 1, what)


def test_bf16_gradients_of_a_whole_views_head(nn):  # noqa: F811
    """A view of 1297 x 840: a pixel's share of the mean loss is 3e-7 of O.  Every
    parameter's gradient in bf16 is near the float32 one: a pixel's gradient
    passes some 20 roundings of 2^-8, which may add up (0.08) where a parameter's
    gradient is mostly one sum over pixels."""
    from msplat_amd.appearance import AppearanceHead
    g = torch.Generator(device="cuda").manual_seed(1)
    view = torch.rand(840, 1297, 3, generator=g, device="cuda")
    head = AppearanceHead(1, dtype=torch.float32)
    head.out.data.normal_(generator=g, std=3e-3)   # what a step leaves
    grads = []
    for dtype in (torch.float32, torch.bfloat16):
        head.dtype = dtype
        loss = (head(view, 0, training=True) - view * 0.8).abs().mean()
        grads.append(torch.autograd.grad(loss, head.parameters()))
    for want, got in zip(*grads):
        assert float(want.norm()) > 0 and float((got - want).norm() / want.norm()) < 0.08
    head.dtype = torch.float16
    with torch.no_grad():
        half = head(view, 0)
        head.dtype = torch.float32
        # the correction, of the size of O, in some 20 roundings of 2^-11
        assert float((half - head(view, 0)).norm()) < 0.01 * float((half - view).norm())
