"""Learned-head operators on the GPU against their formulas in 64 bits.

The tolerances are nn_oracle's elementwise bounds on rounding, derived from
the arithmetic; dropout is equal bit for bit.
"""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import nn_oracle as orc  # noqa: E402

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def nn():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from msplat_amd import nn as module
    return module


def _normal(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=g)).to(dtype).cuda()


def _strided(t, extra, shift):
    """t's values in rows `extra` elements longer, from element `shift` on."""
    rows, dim = t.shape
    buf = torch.full((rows, dim + extra), float("nan"), dtype=t.dtype, device=t.device)
    view = buf[:, shift:shift + dim]
    view.copy_(t)
    return view


NORM_SIZES = [(1, 1), (3, 2), (257, 45), (1000, 64), (70, 100), (33, 256), (19, 511), (9, 1030), (5, 2048), (4, 4097),
              (3, 8192), (5000, 7), (2100, 16)]


@pytest.mark.parametrize("rows,dim", NORM_SIZES)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_layer_norm(nn, dtype, rows, dim):
    x = _normal(1, rows, dim, dtype=dtype, scale=2.0) + _normal(2, rows, 1, dtype=dtype)
    w, b = 1 + _normal(3, dim, dtype=dtype, scale=0.1), _normal(4, dim, dtype=dtype)
    y, mean, rstd = nn.layer_norm_forward(x, w, b, 1e-5)
    want, bound = orc.layer_norm(x, w, b, 1e-5)
    for got, v, e, what in zip((y, mean, rstd), want, bound, ("y", "mean", "rstd")):
        orc.within(got, v, e, f"{what} {rows}x{dim}")
    dy = _normal(5, rows, dim, dtype=dtype)
    got = nn.layer_norm_backward(dy, x, w, mean, rstd)
    want, bound = orc.layer_norm_grad(dy, x, w, mean, rstd)
    for g, v, e, what in zip(got, want, bound, ("dx", "dweight", "dbias")):
        assert g.dtype is dtype
        orc.within(g, v, e, f"{what} {rows}x{dim}")
    again = nn.layer_norm_backward(dy, x, w, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("dim", [45, 64, 600])
def test_layer_norm_without_weight_strided_and_in_place(nn, dim):
    from msplat_amd import _abi
    import ctypes
    x = _normal(7, 130, dim)
    ones, zeros = torch.ones(dim, device="cuda"), torch.zeros(dim, device="cuda")
    y, mean, rstd = nn.layer_norm_forward(x, ones, zeros)
    for extra, shift in ((3, 1), (8, 4)):
        xs, dys = _strided(x, extra, shift), _strided(_normal(8, 130, dim), extra, shift)
        y2, m2, r2 = nn.layer_norm_forward(xs)
        assert torch.equal(y2, y) and torch.equal(m2, mean) and torch.equal(r2, rstd)
        got = nn.layer_norm_backward(dys, xs, None, mean, rstd)
        want = nn.layer_norm_backward(dys.contiguous(), x, ones, mean, rstd)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        # y over x itself
        a = _abi.LayerNormArgs(None, 130, dim, 0, xs.data_ptr(), xs.stride(0), None, None, 1e-5, xs.data_ptr(),
                               xs.stride(0), None, None)
        torch.cuda.synchronize()
        _abi.check(_abi.load().msplat_hip_layer_norm(ctypes.byref(a)))
        torch.cuda.synchronize()
        assert torch.equal(xs, y)
        whole = xs._base
        assert torch.isnan(whole[:, :shift]).all() and torch.isnan(whole[:, shift + dim:]).all()


def test_layer_norm_rows_do_not_mix(nn):
    x = _normal(9, 40, 45)
    clean, _, _ = nn.layer_norm_forward(x)
    x[11, 3], x[12, 44], x[13] = float("nan"), float("inf"), 5.0
    y, _, rstd = nn.layer_norm_forward(x)
    assert torch.isnan(y[11]).all() and torch.isnan(y[12]).any()
    assert (y[13] == 0).all() and abs(float(rstd[13]) - 1e-5 ** -0.5) < 1e-3   # a constant row
    keep = torch.ones(40, dtype=torch.bool)
    keep[11:14] = False
    assert torch.equal(y[keep], clean[keep])


def test_layer_norm_of_a_large_offset(nn):
    """A mean of 1000 standard deviations: the variance does not cancel."""
    x = _normal(10, 64, 200) + 1000.0
    (y, mean, rstd), bound = orc.layer_norm(x, torch.ones(200), torch.zeros(200), 1e-5)
    got = nn.layer_norm_forward(x)
    for g, v, e, what in zip(got, (y, mean, rstd), bound, ("y", "mean", "rstd")):
        orc.within(g, v, e, what)


FFN_SIZES = [(1, 1, 1), (5, 3, 2), (64, 32, 32), (257, 45, 100), (130, 64, 256), (300, 96, 250), (100, 128, 96),
             (77, 130, 40), (90, 200, 333), (65, 256, 64), (33, 250, 1100), (2500, 16, 24), (1300, 48, 192),
             (1, 64, 5000), (40, 143, 946), (4100, 20, 700),
             (30, 70, 3), (4200, 250, 70)]


def _ffn_operands(rows, dim, hidden, dtype, seed=20):
    x = _normal(seed, rows, dim, dtype=dtype)
    wg = _normal(seed + 1, hidden, dim, dtype=dtype, scale=dim ** -0.5)
    wu = _normal(seed + 2, hidden, dim, dtype=dtype, scale=dim ** -0.5)
    wd = _normal(seed + 3, dim, hidden, dtype=dtype, scale=hidden ** -0.5)
    return x, wg, wu, wd


@pytest.mark.parametrize("rows,dim,hidden", FFN_SIZES)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gated_ffn(nn, dtype, rows, dim, hidden):
    for act in ("silu", "gelu"):
        ops = _ffn_operands(rows, dim, hidden, dtype)
        want, bound = orc.gated_ffn_bounds(*ops, act)
        orc.within(nn.gated_ffn_forward(*ops, act), want, bound, f"y {act}")
        dy = _normal(30, rows, dim, dtype=dtype)
        got = nn.gated_ffn_backward(dy, *ops, act)
        want, bound = orc.gated_ffn_grad_bounds(dy, *ops, act)
        for g, v, e, what in zip(got, want, bound, ("dx", "dw_gate", "dw_up", "dw_down")):
            assert g.dtype is dtype
            orc.within(g, v, e, f"{what} {act}")
        again = nn.gated_ffn_backward(dy, *ops, act)
        assert all(torch.equal(p, q) for p, q in zip(got, again))


# more rows than workgroups that take all hidden units: weights through LDS,
# whole (narrow blocks) or block by block, the last with a short last round
FFN_MANY = [(16500, 5, 9), (17001, 32, 600), (20011, 45, 100), (16399, 64, 1000), (9007, 96, 64), (8707, 128, 96),
            (8300, 200, 333), (8201, 256, 40), (65543, 200, 72),
            (131079, 112, 33)]


@pytest.mark.parametrize("rows,dim,hidden", FFN_MANY)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gated_ffn_of_many_rows(nn, dtype, rows, dim, hidden):
    act = "gelu" if dim % 2 else "silu"
    ops = _ffn_operands(rows, dim, hidden, dtype)
    want, bound = orc.gated_ffn_bounds(*ops, act)
    orc.within(nn.gated_ffn_forward(*ops, act), want, bound, f"y {act}")
    dy = _normal(30, rows, dim, dtype=dtype)
    got = nn.gated_ffn_backward(dy, *ops, act)
    want, bound = orc.gated_ffn_grad_bounds(dy, *ops, act)
    for g, v, e, what in zip(got, want, bound, ("dx", "dw_gate", "dw_up", "dw_down")):
        orc.within(g, v, e, f"{what} {act}")
    again = (nn.gated_ffn_forward(*ops, act), *nn.gated_ffn_backward(dy, *ops, act))
    assert all(torch.equal(p, q) for p, q in zip(again, (nn.gated_ffn_forward(*ops, act), *got)))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gated_ffn_errors_are_those_of_rounding(nn, dtype):
    """Whole outputs: h, dg and du are rounded to the type once and the output
    once, each relative uT / sqrt(3) on average, so an output's error in the
    mean square stays below three roundings (float32: below its sums' walk of
    sqrt(n) additions, n the longest sum, and ten roundings)."""
    rows, dim, hidden = 4000, 64, 256
    ops = _ffn_operands(rows, dim, hidden, dtype)
    dy = _normal(30, rows, dim, dtype=dtype)
    got = (nn.gated_ffn_forward(*ops), *nn.gated_ffn_backward(dy, *ops))
    want = (orc.gated_ffn_bounds(*ops, "silu")[0], *orc.gated_ffn_grad_bounds(dy, *ops, "silu")[0])
    uT = orc.UT[dtype][0]
    most = 3 * uT if dtype is not torch.float32 else (rows ** 0.5 + 10) * uT
    for g, v in zip(got, want):
        assert float((g.double().cpu() - v).norm() / v.norm()) < most


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gated_ffn_strides(nn, dtype):
    ops = _ffn_operands(70, 45, 50, dtype)
    dy = _normal(31, 70, 45, dtype=dtype)
    y, grads = nn.gated_ffn_forward(*ops), nn.gated_ffn_backward(dy, *ops)
    for extra, shift in ((3, 1), (11, 5)):
        views = [_strided(t, extra, shift) for t in ops]
        assert torch.equal(nn.gated_ffn_forward(*views), y)
        got = nn.gated_ffn_backward(_strided(dy, extra, shift), *views)
        assert all(torch.equal(p, q) for p, q in zip(got, grads))
    # transposed weights, rows over two axes
    views = [ops[0].view(7, 10, 45), ops[1].t().contiguous().t(), ops[2].t().contiguous().t(),
             ops[3].t().contiguous().t()]
    assert torch.equal(nn.gated_ffn_forward(*views), y.view(7, 10, 45))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gated_ffn_rows_do_not_mix(nn, dtype):
    ops = _ffn_operands(100, 40, 64, dtype)
    dy = _normal(32, 100, 40, dtype=dtype)
    clean, dclean = nn.gated_ffn_forward(*ops), nn.gated_ffn_backward(dy, *ops)[0]
    x = ops[0].clone()
    x[17, 5], x[18, 39] = float("nan"), float("inf")
    y, dx = nn.gated_ffn_forward(x, *ops[1:]), nn.gated_ffn_backward(dy, x, *ops[1:])[0]
    keep = torch.ones(100, dtype=torch.bool)
    keep[17:19] = False
    assert torch.isnan(y[17]).all() and torch.isnan(dx[17]).all()
    assert torch.equal(y[keep], clean[keep]) and torch.equal(dx[keep], dclean[keep])


def test_gated_ffn_of_saturated_gates(nn):
    """Gates of +-200: the sigmoid is 0 or 1 exactly, and no NaN comes of it."""
    x = torch.tensor([[200.0], [-200.0], [0.0]], device="cuda")
    one = torch.ones(1, 1, device="cuda")
    for act in ("silu", "gelu"):
        y = nn.gated_ffn_forward(x, one, one, one, act).flatten().tolist()
        assert y == [40000.0, 0.0, 0.0]
        dx, dg, du, dd = nn.gated_ffn_backward(torch.ones_like(x), x, one, one, one, act)
        assert dx.flatten().tolist() == [400.0, 0.0, 0.0]
        assert float(dd) == 40000.0


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_empty_rows(nn, dtype):
    _, wg, wu, wd = _ffn_operands(1, 40, 24, dtype)
    x = torch.empty(0, 40, dtype=dtype, device="cuda")
    assert nn.gated_ffn_forward(x, wg, wu, wd).shape == (0, 40)
    dx, *grads = nn.gated_ffn_backward(x, x, wg, wu, wd)
    assert dx.shape == (0, 40) and all((g == 0).all() for g in grads)
    w = torch.ones(40, dtype=dtype, device="cuda")
    y, mean, rstd = nn.layer_norm_forward(x, w, w)
    assert y.shape == (0, 40) and mean.shape == (0,)
    dx, dw, db = nn.layer_norm_backward(x, x, w, mean, rstd)
    assert dx.shape == (0, 40) and (dw == 0).all() and (db == 0).all()
    assert nn.dropout_add_forward(x, x, 0.5, 1, 2).shape == (0, 40)


@pytest.mark.parametrize("rows,dim", [(1, 1), (257, 45), (1000, 64), (37, 1030), (4, 9000)])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_dropout_add(nn, dtype, rows, dim):
    x, r = _normal(40, rows, dim, dtype=dtype), _normal(41, rows, dim, dtype=dtype)
    for p in (0.0, 0.1, 0.5, 1.0):
        seed, offset = 0xFEDCBA9876543210, 0x1122334455667788
        want = orc.dropout_add(x, r, p, seed, offset)
        assert torch.equal(nn.dropout_add_forward(x, r, p, seed, offset).cpu(), want), p
        assert torch.equal(nn.dropout_add_backward(x, p, seed, offset).cpu(), orc.dropout_add(x, None, p, seed, offset)), p
    views = [_strided(t, 5, 3) for t in (x, r)]
    assert torch.equal(nn.dropout_add_forward(*views, 0.1, 5, 6), nn.dropout_add_forward(x, r, 0.1, 5, 6))


def test_dropped_elements_count_as_zero(nn):
    x = torch.full((64, 45), float("nan"), device="cuda")
    keep = orc.keep_mask(64, 45, 0.5, 3, 4).cuda()
    y = nn.dropout_add_forward(x, torch.ones_like(x), 0.5, 3, 4)
    assert torch.isnan(y[keep]).all() and (y[~keep] == 1).all()


def _block(nn, x, w, b, wg, wu, wd, step):
    return nn.dropout_add(nn.gated_ffn(nn.layer_norm(x, w, b), wg, wu, wd, "gelu"), x, 0.25, 11, step)


def _block64(x, w, b, wg, wu, wd, step):
    d = x - x.mean(1, keepdim=True)
    n = d * (d.square().mean(1, keepdim=True) + 1e-5).rsqrt() * w + b
    keep = orc.keep_mask(x.shape[0], x.shape[1], 0.25, 11, step)
    return x + torch.where(keep, orc.gated_ffn(n, wg, wu, wd, "gelu") / 0.75, 0.0)


def test_a_block_and_its_gradients(nn):
    """The three together by autograd, in float32: against the 64-bit block,
    its gradients and a central difference along a random direction.  The
    chain is some 300 roundings long per output, of terms of its own size."""
    rows, dim, hidden = 200, 48, 100
    x, wg, wu, wd = _ffn_operands(rows, dim, hidden, torch.float32)
    w, b = 1 + _normal(50, dim, scale=0.1), _normal(51, dim, scale=0.1)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, wg, wu, wd)]
    dy = _normal(52, rows, dim)
    y = _block(nn, *leaves, 3)
    got = torch.autograd.grad(y, leaves, dy)
    wide = [t.detach().double().cpu().requires_grad_() for t in leaves]
    y64 = _block64(*wide, 3)
    want = torch.autograd.grad(y64, wide, dy.double().cpu())
    for g, v in zip((y.detach(), *got), (y64.detach(), *want)):
        assert float((g.double().cpu() - v).norm() / v.norm()) < 300 * orc.U
    way = [torch.randn(t.shape, generator=torch.Generator().manual_seed(60 + i), dtype=torch.float64)
           for i, t in enumerate(wide)]
    h = 1e-5
    up, down = (((_block64(*[t.detach() + s * h * v for t, v in zip(wide, way)], 3)) * dy.double().cpu()).sum()
                for s in (1, -1))
    along = sum((g.double().cpu() * v).sum() for g, v in zip(got, way))
    size = sum((g.double().cpu() * v).abs().sum() for g, v in zip(got, way))
    # the difference's own error is of order h^2 = 1e-10
    assert abs(float((up - down) / (2 * h) - along)) < float(size) * 1e-6


def test_expanded_gradients(nn):
    """The gradients of sums reach the operators as expanded tensors, whose
    rows or elements are one in memory."""
    x, wg, wu, wd = (t.requires_grad_() for t in _ffn_operands(50, 40, 60, torch.float32))
    r = _normal(61, 50, 40).requires_grad_()
    w = (1 + _normal(62, 40, scale=0.1)).requires_grad_()
    v = _normal(63, 40)
    for loss in (lambda y: y.sum(), lambda y: (y.sum(0) * v).sum()):
        y = nn.dropout_add(nn.gated_ffn(nn.layer_norm(x, w), wg, wu, wd), r, 0.25, 5, 6)
        leaves = (x, wg, wu, wd, w, r)
        got = torch.autograd.grad(loss(y), leaves)
        y = nn.dropout_add(nn.gated_ffn(nn.layer_norm(x, w), wg, wu, wd), r, 0.25, 5, 6)
        ones = torch.ones_like(y)
        dy = ones if torch.equal(torch.autograd.grad(loss(r * 1), r)[0], ones) else v.expand(50, 40).contiguous()
        want = torch.autograd.grad(y, leaves, dy)
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_offsets_beyond_32_bits(nn, dtype):
    """60000 rows 40000 elements apart: the last ones start past 2^31 elements."""
    rows, dim, stride = 60000, 40, 40000
    buf = torch.empty((rows - 1) * stride + dim, dtype=dtype, device="cuda")

    def far(t):
        view = buf.as_strided((rows, dim), (stride, 1))
        view.copy_(t)
        return view

    x, wg, wu, wd = _ffn_operands(rows, dim, 48, dtype)
    w = torch.ones(dim, dtype=dtype, device="cuda")
    y, mean, rstd = nn.layer_norm_forward(x, w, w)
    for call in (lambda t: nn.layer_norm_forward(t, w, w), lambda t: nn.layer_norm_backward(x, t, w, mean, rstd),
                 lambda t: nn.layer_norm_backward(t, x, w, mean, rstd),
                 lambda t: (nn.gated_ffn_forward(t, wg, wu, wd),), lambda t: nn.gated_ffn_backward(x, t, wg, wu, wd),
                 lambda t: nn.gated_ffn_backward(t, x, wg, wu, wd), lambda t: (nn.dropout_add_forward(x, t, 0.5, 1, 2),)):
        assert all(torch.equal(p, q) for p, q in zip(call(far(x)), call(x)))


def test_other_streams(nn):
    x, wg, wu, wd = _ffn_operands(3000, 64, 128, torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    want = _block(nn, x, w, w, wg, wu, wd, 9)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                y = _block(nn, x * 1, w, w, wg, wu, wd, 9)
            got.append(y)
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)


def test_graph_replays(nn):
    x, wg, wu, wd = _ffn_operands(500, 64, 128, torch.float16)
    dy = _normal(70, 500, 64, dtype=torch.float16)
    w = torch.ones(64, dtype=torch.float16, device="cuda")

    def step():
        n, mean, rstd = nn.layer_norm_forward(x, w, w)
        y = nn.dropout_add_forward(nn.gated_ffn_forward(n, wg, wu, wd), x, 0.1, 1, 2)
        dn, *grads = nn.gated_ffn_backward(dy, n, wg, wu, wd)
        return [y, *grads, *nn.layer_norm_backward(dn, x, w, mean, rstd)]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        x.copy_(_normal(80 + k, 500, 64, dtype=torch.float16))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), k


def test_python_checks(nn):
    x = _normal(90, 8, 16)
    w = _normal(91, 24, 16)
    with pytest.raises(ValueError, match="w_up"):
        nn.gated_ffn_forward(x, w, w[:, :8], w.t())
    with pytest.raises(ValueError, match="w_down"):
        nn.gated_ffn_forward(x, w, w, w)
    with pytest.raises(ValueError, match="activation"):
        nn.gated_ffn_forward(x, w, w, w.t(), "relu")
    with pytest.raises(ValueError, match="float16"):
        nn.gated_ffn_forward(x, w.half(), w, w.t())
    with pytest.raises(ValueError, match="none of"):
        nn.layer_norm_forward(x.double())
    with pytest.raises(ValueError, match="weight"):
        nn.layer_norm_forward(x, torch.ones(15, device="cuda"))
    with pytest.raises(ValueError, match="dy"):
        nn.gated_ffn_backward(x[:5], x, w, w, w.t())
    with pytest.raises(ValueError, match="residual"):
        nn.dropout_add_forward(x, x[:, :8], 0.1, 1, 2)
    with pytest.raises(ValueError, match="outside"):
        nn.dropout_add_forward(x, None, 1.5, 1, 2)
    from msplat_amd._abi import MsplatError
    wide = _normal(92, 4, 300)
    with pytest.raises(MsplatError, match="dim 300"):
        nn.gated_ffn_forward(wide, _normal(93, 8, 300), _normal(94, 8, 300), _normal(95, 300, 8))
