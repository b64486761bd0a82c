"""8-bit rows and the root-mean-square norm on the GPU against their formulas in
64 bits.  Packed rows are equal bit for bit; the norm's tolerances are
more_oracle's elementwise bounds on rounding."""
from __future__ import annotations

import ctypes

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import more_oracle as orc  # noqa: E402
from nn_oracle import within  # noqa: E402
from test_gpu_nn import DTYPES, IDS, _normal, _strided, nn  # noqa: E402,F401

SIZES = [(1, 1), (3, 2), (257, 45), (1000, 64), (70, 100), (33, 256), (19, 511), (9, 1030), (5, 2048), (4, 4097),
         (3, 8192), (5000, 7), (2100, 16), (6, 31), (7, 33), (65, 129), (1, 128)]


def _bytes(t):
    return t.view(torch.uint8).cpu()


def _same(a, b):
    """Equal values, NaN where the other has NaN (a type's largest may have become infinite, and NaN in 8 bits)."""
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0))


def _check_packed(m, x, what):
    """Every byte of m against packing x."""
    values, codes = orc.mx8(x)
    rows, dim = x.shape
    n = codes.shape[1]
    scales = m.scales.cpu().to(torch.int64).view(rows, -1)
    assert torch.equal(scales[:, :n], codes), f"{what}: scales"
    assert (scales[:, n:] == 0).all()
    data = m.data.cpu().view(torch.float8_e4m3fn).view(rows, -1)
    assert (_bytes(data)[:, dim:] == 0).all(), f"{what}: padding"
    s = torch.exp2(codes.double() - 127).repeat_interleave(32, 1)[:, :dim]
    got = data[:, :dim].double() * s
    assert _same(got, values), f"{what}: elements"
    return values


@pytest.mark.parametrize("rows,dim", SIZES + [(2, 20000)])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_packed_rows(nn, dtype, rows, dim):
    x = (_normal(1, rows, dim) * torch.exp2(4 * _normal(2, rows, dim))).to(dtype)
    for view in (x, _strided(x, 5, 3)):
        m = nn.mx8_pack(view)
        assert m.shape == x.shape and m.dtype is dtype
        values = _check_packed(m, x, f"{rows}x{dim}")
        back = nn.mx8_unpack(m)
        assert back.dtype is dtype and _same(back.double().cpu(), values.to(dtype).double())
    assert _same(nn.mx8_unpack(m, torch.float32).double().cpu(), values)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_packed_extremes(nn, dtype):
    """Each in a block of its own, beside ordinary numbers: the largest and least
    numbers of the type, NaN and infinities, blocks of zeros and of NaN alone,
    borders of the scale and ties of the rounding."""
    info = torch.finfo(dtype)
    nan, inf = float("nan"), float("inf")
    rows = [[info.max, 1.0], [-info.max, info.max], [info.tiny, -info.tiny], [info.smallest_normal / 8, 0.0],
            [nan, 3.0, -5.0], [inf, 2.0, -inf, 7.0], [0.0] * 32, [nan] * 32, [448.0, 17.0, 18.0, 19.0],
            [448.5, 17.0, 1.0], [896.0, 1.0], [900.0, 1.0], [1.75, 1.0625, 1.1875, -1.0625], [61440.0, 61441.0, -64000.0],
            [-0.0, 1.0], [2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -10, 256.0]]
    x = torch.zeros(len(rows), 32)
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r)
    x = x.to(dtype).cuda()
    for shaped in (x, x.reshape(4, -1), x.reshape(1, -1)):
        values = _check_packed(nn.mx8_pack(shaped), shaped, str(shaped.shape))
        back = nn.mx8_unpack(nn.mx8_pack(shaped)).double().cpu()
        assert _same(back, values.to(dtype).double())
        assert not torch.isinf(back).any()


@pytest.mark.parametrize("mx", [False, True], ids=["plain", "mx8"])
@pytest.mark.parametrize("rows,dim", SIZES)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rms_norm(nn, dtype, rows, dim, mx):
    x = _normal(1, rows, dim, dtype=dtype, scale=2.0) + _normal(2, rows, 1, dtype=dtype)
    w, r = 1 + _normal(3, dim, dtype=dtype, scale=0.1), _normal(4, rows, dim, dtype=dtype)
    for residual in (r, None):
        y, total, rstd = nn.rms_norm_forward(x, w, residual, 1e-5, mx8=mx)
        if residual is None:
            assert total is x
        else:
            assert torch.equal(total, (x.float() + r.float()).to(dtype))
        want, want_rstd, e_32, e_y, e_rstd = orc.rms_norm(total, w, 1e-5)
        within(rstd, want_rstd, e_rstd, f"rstd {rows}x{dim}")
        if mx:
            within(nn.mx8_unpack(y, torch.float32), want, orc.mx8_bound(want, e_32), f"y in mx8 {rows}x{dim}")
            assert (_bytes(y.data).view(rows, -1)[:, dim:] == 0).all()
        else:
            within(y, want, e_y, f"y {rows}x{dim}")
    total = x
    dy, dt = _normal(5, rows, dim, dtype=dtype), _normal(6, rows, dim, dtype=dtype)
    kept = nn.mx8_pack(total) if mx else total
    values = nn.mx8_unpack(kept, torch.float32) if mx else total
    for dtotal in (dt, None):
        got = nn.rms_norm_backward(dy, kept, w, rstd, dtotal)
        want, bound = orc.rms_norm_grad(dy, values, w, rstd, dtotal)
        for g, v, e, what in zip(got, want, bound, ("dx", "dweight")):
            assert g.dtype is dtype
            within(g, v, e, f"{what} {rows}x{dim}")
        again = nn.rms_norm_backward(dy, kept, w, rstd, dtotal)
        assert all(torch.equal(p, q) for p, q in zip(got, again))
    dx, none = nn.rms_norm_backward(dy, kept, w, rstd, dtotal, wanted=(True, False))
    assert none is None and torch.equal(dx, got[0])
    none, dw = nn.rms_norm_backward(dy, kept, w, rstd, dtotal, wanted=(False, True))
    assert none is None and torch.equal(dw, got[1])


@pytest.mark.parametrize("dim", [45, 64, 600, 2100])
def test_rms_norm_strided_and_in_place(nn, dim):
    from msplat_amd import _abi
    rows = 130
    x, r, dy = _normal(7, rows, dim), _normal(8, rows, dim), _normal(9, rows, dim)
    ones = torch.ones(dim, device="cuda")
    y, total, rstd = nn.rms_norm_forward(x, ones, r)
    dx, dw = nn.rms_norm_backward(dy, total, ones, rstd, r)
    for extra, shift in ((3, 1), (8, 4)):
        xs, rs, dys, ts = (_strided(t, extra, shift) for t in (x, r, dy, total))
        got = nn.rms_norm_forward(xs, None, rs)
        assert all(torch.equal(p, q) for p, q in zip(got, (y, total, rstd)))
        got = nn.rms_norm_backward(dys, ts, None, rstd, rs)
        assert torch.equal(got[0], dx) and torch.equal(got[1], dw)
        # y over x and the sum over the residual; then dx over dy
        a = _abi.RmsNormArgs(None, rows, dim, 0, xs.data_ptr(), xs.stride(0), rs.data_ptr(), rs.stride(0), None, 1e-5,
                             xs.data_ptr(), xs.stride(0), None, rs.data_ptr(), rs.stride(0), None)
        torch.cuda.synchronize()
        _abi.check(_abi.load().msplat_hip_rms_norm(ctypes.byref(a)))
        torch.cuda.synchronize()
        assert torch.equal(xs, y) and torch.equal(rs, total)
        g = _abi.RmsNormGradArgs(None, rows, dim, 0, dys.data_ptr(), dys.stride(0), None, 0, total.data_ptr(), dim, None,
                                 None, rstd.data_ptr(), dys.data_ptr(), dys.stride(0), None, None, 0)
        _abi.check(_abi.load().msplat_hip_rms_norm_backward(ctypes.byref(g)))
        torch.cuda.synchronize()
        assert torch.equal(dys, nn.rms_norm_backward(dy, total, None, rstd)[0])
        for t in (xs, rs, dys):
            assert torch.isnan(t._base[:, :shift]).all() and torch.isnan(t._base[:, shift + dim:]).all()


def test_rows_do_not_mix(nn):
    x = _normal(10, 40, 45)
    clean = nn.rms_norm_forward(x)[0]
    x[11, 3], x[12, 44], x[13] = float("nan"), float("inf"), 0.0
    y, _, rstd = nn.rms_norm_forward(x)
    assert torch.isnan(y[11]).all() and torch.isnan(y[12, 44]) and (y[12, :44] == 0).all()
    assert (y[13] == 0).all() and abs(float(rstd[13]) - 1e-5 ** -0.5) < 1e-3
    keep = torch.ones(40, dtype=torch.bool)
    keep[11:14] = False
    assert torch.equal(y[keep], clean[keep])
    m = nn.mx8_unpack(nn.rms_norm_forward(x, mx8=True)[0])
    assert torch.isnan(m[11]).all() and torch.isfinite(m[keep]).all() and (m[13] == 0).all()
    # zeros with no eps: 0 * infinity, NaN in every element of the row, none behind its end
    zero = nn.rms_norm_forward(torch.zeros(3, 45, device="cuda"), eps=0.0, mx8=True)[0]
    assert torch.isnan(nn.mx8_unpack(zero)).all() and (_bytes(zero.data)[:, 45:] == 0).all()


def test_no_rows(nn):
    x = torch.empty(0, 45, device="cuda")
    y, total, rstd = nn.rms_norm_forward(x, None, x)
    assert y.shape == (0, 45) and total.shape == (0, 45) and rstd.shape == (0,)
    dx, dw = nn.rms_norm_backward(x, x, None, rstd)
    assert dx.shape == (0, 45) and (dw == 0).all()
    m = nn.mx8_pack(x)
    assert m.shape == (0, 45) and nn.mx8_unpack(m).shape == (0, 45)
    assert nn.rms_norm_forward(x, mx8=True)[0].shape == (0, 45)


@pytest.mark.parametrize("checkpoint", [None, "mx8"])
def test_autograd(nn, checkpoint):
    """Against torch's own differentiation of the formula in 64 bits, the sum
    replaced by what the checkpoint holds; shared and broadcast inputs."""
    x0 = _normal(11, 4, 6, 45).cpu()
    r0 = _normal(12, 45).cpu()
    w0 = (1 + 0.1 * _normal(13, 45)).cpu()
    x, w = x0.cuda().requires_grad_(), w0.cuda().requires_grad_()
    r = r0.cuda().requires_grad_()
    y, total = nn.rms_norm(x, w, r.expand(4, 6, 45), checkpoint=checkpoint)
    again = nn.rms_norm(total, w, checkpoint=checkpoint)
    (y.square().sum() + (again * total).sum() + 0.5 * total.sum()).backward()

    def kept(t):
        if checkpoint is None:
            return t
        packed = orc.mx8(t.detach().float().reshape(-1, 45))[0].reshape(t.shape)
        return t + (packed - t.detach())

    # with a checkpoint the gradient is that at the packed sum, with the forward's rstd, of the forward's y
    xd, rd, wd = (t.double().requires_grad_() for t in (x0, r0, w0))
    t = xd + rd
    td = t.detach()

    def norm_grad(dy, dtotal):
        rstd = (td.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        n = kept(td) * rstd
        g = dy * wd.detach()
        return rstd * (g - n * (g * n).mean(-1, keepdim=True)) + dtotal, (dy * n).sum((0, 1))

    rstd = (td.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    yd = td * rstd * wd.detach()
    d2, dw2 = norm_grad(td, torch.zeros_like(td))           # again * total, by again
    d1, dw1 = norm_grad(2 * yd, d2 + yd + 0.5)              # and by total, and total's own
    for got, want in ((x.grad, d1), (r.grad, d1.sum((0, 1))), (w.grad, dw1 + dw2)):
        assert (got.double().cpu() - want).abs().max() < 1e-4 * want.abs().max()
    y, total = nn.rms_norm(x, w, r.expand(4, 6, 45), checkpoint=checkpoint)
    gx, gw = torch.autograd.grad(total.sum(), (x, w))       # y unused
    assert (gx == 1).all() and (gw == 0).all()


def test_far_offsets(nn):
    """Rows whose elements lie beyond 2^32 bytes and 2^31 elements."""
    stride = (1 << 30) + 8
    buf = torch.empty(3 * stride + 64, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(buf, (4, 50), (stride, 1))
    small = _normal(14, 4, 50, dtype=torch.bfloat16)
    x.copy_(small)
    y, _, rstd = nn.rms_norm_forward(x)
    y0, _, rstd0 = nn.rms_norm_forward(small)
    assert torch.equal(y, y0) and torch.equal(rstd, rstd0)
    assert torch.equal(nn.rms_norm_backward(x, x, None, rstd)[0], nn.rms_norm_backward(small, small, None, rstd)[0])
    p, q = nn.mx8_pack(x), nn.mx8_pack(small)
    assert torch.equal(_bytes(p.data), _bytes(q.data)) and torch.equal(p.scales, q.scales)
    del buf, x
    # 2^32 bytes of packed rows and more
    rows = (1 << 32) // 64 + 5
    x = torch.zeros(rows, 40, dtype=torch.bfloat16, device="cuda")
    x[-3:] = _normal(15, 3, 40, dtype=torch.bfloat16)
    m = nn.mx8_pack(x)
    tail = nn.mx8_pack(x[-3:].clone())
    assert torch.equal(_bytes(m.data[-3:]), _bytes(tail.data)) and torch.equal(m.scales[-3:], tail.scales)
    assert torch.equal(nn.mx8_unpack(m)[-3:], nn.mx8_unpack(tail))
    y = nn.rms_norm_forward(x, mx8=True)[0]
    want = nn.rms_norm_forward(x[-3:].clone(), mx8=True)[0]
    assert torch.equal(_bytes(y.data[-3:]), _bytes(want.data))


def test_streams_and_replays(nn):
    """On a stream of its own, and in a captured graph whose replays see new inputs."""
    x, r, dy = (_normal(s, 300, 100, dtype=torch.bfloat16) for s in (16, 17, 18))
    w = 1 + _normal(19, 100, dtype=torch.bfloat16, scale=0.1)

    def step():
        y, total, rstd = nn.rms_norm_forward(x, w, r)
        m, _, _ = nn.rms_norm_forward(total, w, mx8=True)
        kept = nn.mx8_pack(total)
        return (y, total, rstd, nn.mx8_unpack(m), *nn.rms_norm_backward(dy, kept, w, rstd, y))

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (20, 21, 22):
        for t in (x, r, dy):
            t.copy_(_normal(seed + t.data_ptr() % 7, 300, 100, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(p, q) for p, q in zip(got, step()))
