"""The linear layer on the GPU against its formulas in 64 bits, within
more_oracle's elementwise bounds on rounding."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import more_oracle as orc  # noqa: E402
from linear_sizes import FEW, ONE_PASS, RESIDENT, SIZES, STREAMED  # noqa: E402
from test_gpu_nn import DTYPES, IDS, _normal, _strided, nn  # noqa: E402,F401

ACTS = [None, "silu", "gelu"]


def _operands(rows, inner, outer, dtype, seed=30):
    x = _normal(seed, rows, inner, dtype=dtype)
    w = _normal(seed + 1, outer, inner, dtype=dtype, scale=inner ** -0.5)
    b = _normal(seed + 2, outer, dtype=dtype, scale=0.3)
    return x, w, b


def _check_forward(got, x, w, b, r, act, out_dtype, what):
    y, z, e_y, _ = orc.linear(x, w, b, r, act, out_dtype)
    assert got.dtype is out_dtype
    orc.near(got, y, e_y, what)


@pytest.mark.parametrize("rows,inner,outer", SIZES + FEW + RESIDENT + STREAMED)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_forward(nn, dtype, rows, inner, outer):
    x, w, b = _operands(rows, inner, outer, dtype)
    for i, act in enumerate(ACTS):
        out_dtype = DTYPES[(DTYPES.index(dtype) + i) % 3] if act else dtype
        r = _normal(40, rows, outer, dtype=out_dtype)
        y, z = nn.linear_forward(x, w, b, r, act, out_dtype, keep=True)
        _check_forward(y, x, w, b, r, act, out_dtype, f"y {act}")
        _, want, _, e_z = orc.linear(x, w, b, None, None, dtype)
        uT, tiny = orc.UT[dtype]
        assert z.dtype is dtype
        orc.near(z, want, e_z + (uT + orc.U) * want.abs() + tiny, "z")
        assert torch.equal(nn.linear_forward(x, w, b, r, act, out_dtype), y)
    _check_forward(nn.linear_forward(x, w), x, w, None, None, None, dtype, "product alone")


@pytest.mark.parametrize("rows,inner,outer", FEW + [RESIDENT[1], RESIDENT[7], STREAMED[1], STREAMED[6]])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_forward_of_every_pair_of_types(nn, dtype, rows, inner, outer):
    x, w, b = _operands(rows, inner, outer, dtype)
    for out_dtype in DTYPES:
        for act in ACTS:
            for bias, r in ((b, None), (None, _normal(44, rows, outer, dtype=out_dtype))):
                got = nn.linear_forward(x, w, bias, r, act, out_dtype)
                _check_forward(got, x, w, bias, r, act, out_dtype, f"y {act} in {out_dtype}")


@pytest.mark.parametrize("rows,inner,outer", SIZES + FEW + RESIDENT + STREAMED)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_forward_of_8_bits(nn, dtype, rows, inner, outer):
    """Values of 8 bits multiply exactly, so the bounds are those of 32-bit sums."""
    x, w, _ = _operands(rows, inner, outer, dtype)
    x, w = nn.mx8_pack(x * torch.exp2(3 * _normal(41, rows, 1)).to(dtype)), nn.mx8_pack(w)
    xv, wv = nn.mx8_unpack(x, torch.float32), nn.mx8_unpack(w, torch.float32)
    b, r = _normal(42, outer), _normal(43, rows, outer, dtype=dtype)
    for act in ACTS:
        _check_forward(nn.linear_forward(x, w, b, r, act), xv, wv, b, r, act, dtype, f"y {act}")
    got = nn.linear_forward(x, w, out_dtype=torch.float32)
    _check_forward(got, xv, wv, None, None, None, torch.float32, "in float32")


def _check_backward(nn, dtype, rows, inner, outer, act, mx, out_dtype):
    x, w, _ = _operands(rows, inner, outer, dtype)
    dy = _normal(50, rows, outer, dtype=out_dtype)
    z = _normal(51, rows, outer, dtype=dtype, scale=2.0) if act else None
    xk, zk, xv, zv = x, z, x, z
    if mx:
        xk = nn.mx8_pack(x)
        xv = nn.mx8_unpack(xk)   # the products take x in its own type
        if act:
            zk = nn.mx8_pack(z)
            zv = nn.mx8_unpack(zk, torch.float32)
    got = nn.linear_backward(dy, xk, w, zk, act)
    want, bound = orc.linear_grad(dy, xv, w, zv, act, dtype)
    for g, v, e, what in zip(got, want, bound, ("dx", "dweight", "dbias")):
        assert g.dtype is dtype
        orc.near(g, v, e, f"{what} {act} mx={mx}")
    return (dy, xk, w, zk, act), got


@pytest.mark.parametrize("mx", [False, True], ids=["plain", "mx8"])
@pytest.mark.parametrize("rows,inner,outer", SIZES + FEW + RESIDENT + STREAMED + ONE_PASS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_backward(nn, dtype, rows, inner, outer, mx):
    for i, act in enumerate(ACTS):
        for out_dtype in {dtype, DTYPES[(DTYPES.index(dtype) + i) % 3]}:
            call, got = _check_backward(nn, dtype, rows, inner, outer, act, mx, out_dtype)
            for k in range(3):
                alone = nn.linear_backward(*call, wanted=tuple(j == k for j in range(3)))
                assert all(t is None for j, t in enumerate(alone) if j != k)
                assert torch.equal(alone[k], got[k]), f"gradient {k} by itself"
            assert all(torch.equal(p, q) for p, q in zip(got, nn.linear_backward(*call)))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_strided(nn, dtype):
    rows, inner, outer = 70, 45, 52
    x, w, b = _operands(rows, inner, outer, dtype)
    r, dy, z = (_normal(s, rows, outer, dtype=dtype) for s in (52, 53, 54))
    y = nn.linear_forward(x, w, b, r, "silu")
    grads = nn.linear_backward(dy, x, w, z, "silu")
    for extra, shift in ((3, 1), (8, 4)):
        xs, ws, rs, dys, zs = (_strided(t, extra, shift) for t in (x, w, r, dy, z))
        assert torch.equal(nn.linear_forward(xs, ws, b, rs, "silu"), y)
        got = nn.linear_backward(dys, xs, ws, zs, "silu")
        assert all(torch.equal(p, q) for p, q in zip(got, grads))
    # other orders: a transposed weight, an expanded gradient, more axes
    assert torch.equal(nn.linear_forward(x, w.t().contiguous().t(), b, r, "silu"), y)
    one = dy[:1].expand(rows, outer)
    got = nn.linear_backward(one, x, w, z, "silu")
    want = nn.linear_backward(one.contiguous(), x, w, z, "silu")
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    cube = nn.linear_forward(x.view(7, 10, inner), w, b, r.view(7, 10, outer), "silu")
    assert cube.shape == (7, 10, outer) and torch.equal(cube.view(rows, outer), y)


def test_outputs_end_where_they_do(nn):
    """y over the residual, in rows with strangers around, z beside it."""
    import ctypes
    from msplat_amd import _abi
    rows, inner, outer = 70, 45, 53
    x, w, b = _operands(rows, inner, outer, torch.float32)
    r = _normal(55, rows, outer)
    want = nn.linear_forward(x, w, b, r, "gelu")
    _, z = nn.linear_forward(x, w, b, r, "gelu", keep=True)
    y, zs = _strided(r, 7, 2), _strided(r, 5, 3)
    a = _abi.LinearArgs(None, rows, inner, outer, 0, 0, 1, x.data_ptr(), inner, None, w.data_ptr(), inner, None, b.data_ptr(),
                        y.data_ptr(), y.stride(0), y.data_ptr(), y.stride(0), zs.data_ptr(), zs.stride(0), None, 0)
    ws = torch.empty(max(1, _abi.load().msplat_hip_linear_workspace(rows, inner, outer, 0)), dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.nbytes
    torch.cuda.synchronize()
    _abi.check(_abi.load().msplat_hip_linear(ctypes.byref(a)))
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(zs, z)
    for t, shift in ((y, 2), (zs, 3)):
        assert torch.isnan(t._base[:, :shift]).all() and torch.isnan(t._base[:, shift + outer:]).all()


def test_no_rows(nn):
    x, w = torch.empty(0, 45, device="cuda"), torch.ones(7, 45, device="cuda")
    assert nn.linear_forward(x, w).shape == (0, 7)
    dy = torch.empty(0, 7, device="cuda")
    for z, act in ((None, None), (dy, "gelu")):
        dx, dw, db = nn.linear_backward(dy, x, w, z, act)
        assert dx.shape == (0, 45) and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rows_do_not_mix(nn, dtype):
    x, w, b = _operands(80, 45, 40, dtype)
    clean = nn.linear_forward(x, w, b, None, "silu")
    x[11, 3], x[12, 44], x[13] = float("nan"), float("inf"), 0.0
    y = nn.linear_forward(x, w, b, None, "silu")
    assert torch.isnan(y[11]).all() and not torch.isfinite(y[12]).all()
    keep = torch.ones(80, dtype=torch.bool)
    keep[11:14] = False
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("checkpoint", [None, "mx8"])
@pytest.mark.parametrize("act", ACTS)
def test_autograd(nn, act, checkpoint):
    x0, w0, b0 = _operands(24, 45, 40, torch.float32)
    r0 = _normal(60, 40)
    leaves = [t.clone().requires_grad_() for t in (x0, w0, b0, r0)]
    x, w, b, r = leaves
    y = nn.linear(x.view(4, 6, 45), w, b, r.expand(4, 6, 40), act, checkpoint=checkpoint)
    g = _normal(61, 4, 6, 40)
    y.backward(g)
    z0 = nn.linear_forward(x0, w0, b0)
    xk, zk = (nn.mx8_unpack(nn.mx8_pack(t)) if checkpoint else t for t in (x0, z0))
    (dx, dw, db), bound = orc.linear_grad(g.view(24, 40), xk, w0, zk, act, torch.float32)
    orc.near(x.grad, dx, bound[0], "x")
    orc.near(w.grad, dw, bound[1], "weight")
    orc.near(b.grad, db, bound[2], "bias")
    assert (r.grad - g.sum((0, 1))).abs().max() < 1e-4
    # half of them, with a result in another type
    y = nn.linear(x0, w, None, None, act, torch.bfloat16, checkpoint)
    assert y.dtype is torch.bfloat16
    gw, = torch.autograd.grad(y, (w,), g.view(24, 40).bfloat16())
    assert gw.shape == w.shape and torch.isfinite(gw).all()


def test_far_offsets(nn):
    """Rows whose elements lie beyond 2^32 bytes and 2^31 elements, of every matrix."""
    stride = (1 << 30) + 8
    big = [torch.as_strided(torch.empty(3 * stride + 64, dtype=torch.bfloat16, device="cuda"), (4, 50), (stride, 1))
           for _ in range(3)]
    x, w, b = _operands(4, 50, 50, torch.bfloat16)
    dy = _normal(62, 4, 50, dtype=torch.bfloat16)
    for far, t in zip(big, (x, dy, w[:4])):
        far.copy_(t)
    xs, dys, ws = big
    assert torch.equal(nn.linear_forward(xs, ws, b[:4], None, "gelu"), nn.linear_forward(x, w[:4], b[:4], None, "gelu"))
    y = nn.linear_forward(xs, w, b, dys, "gelu")
    assert torch.equal(y, nn.linear_forward(x, w, b, dy, "gelu"))
    got, want = nn.linear_backward(dys, xs, w, dys, "silu"), nn.linear_backward(dy, x, w, dy, "silu")
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    got, want = nn.linear_backward(dy[:, :4].contiguous(), x, ws), nn.linear_backward(dy[:, :4].contiguous(), x, w[:4].contiguous())
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_streams_and_replays(nn):
    rows, inner, outer = 300, 100, 72
    x, w, b = _operands(rows, inner, outer, torch.bfloat16)
    r, dy = (_normal(s, rows, outer, dtype=torch.bfloat16) for s in (63, 64))

    def step():
        y, z = nn.linear_forward(x, w, b, r, "silu", torch.float32 if r.dtype is torch.float32 else None, keep=True)
        m = nn.linear_forward(nn.mx8_pack(x), nn.mx8_pack(w), None, r)
        return (y, z, m, *nn.linear_backward(dy, nn.mx8_pack(x), w, z, "silu"), *nn.linear_backward(dy, x, w))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (65, 66, 67):
        for i, t in enumerate((x, r, dy)):
            t.copy_(_normal(seed + 10 * i, *t.shape, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(p, q) for p, q in zip(got, step()))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_ends_of_the_activations(nn, dtype):
    """Far arguments: a(v) is v or 0, a'(v) 1 or 0, whatever the powers between overflow to."""
    big = 6e4 if dtype is torch.float16 else 1e30
    v = torch.tensor([big, -big, 100.0, -100.0, 0.0, 30.0, -30.0], dtype=dtype, device="cuda")[:, None]
    one = torch.ones(1, 1, dtype=dtype, device="cuda")
    for act in ("silu", "gelu"):
        y, z = nn.linear_forward(v, one, activation=act, keep=True)
        assert torch.equal(z, v)
        want = torch.where(v > 0, v, torch.zeros_like(v))
        assert float((y - want).abs().max()) < 1e-8
        dx, _, _ = nn.linear_backward(torch.ones_like(v), v, one, z, act)
        want = torch.where(v > 0, 1.0, torch.where(v == 0, 0.5, 0.0))
        assert float((dx.float() - want).abs().max()) < 1e-8


def test_rows_with_infinities_and_a_tail(nn):
    """A width that no piece divides, in every kernel: an infinity stays in its row."""
    for rows, inner, outer in ((40, 45, 40), (70000, 45, 40), (70000, 300, 40)):
        x, w, b = _operands(rows, inner, outer, torch.bfloat16)
        clean = nn.linear_forward(x, w, b)
        x[7, inner - 1], x[8, 0] = float("inf"), float("nan")
        y = nn.linear_forward(x, w, b)
        keep = torch.ones(rows, dtype=torch.bool, device="cuda")
        keep[7:9] = False
        assert torch.equal(y[keep], clean[keep]) and not torch.isfinite(y[7]).any() and torch.isnan(y[8]).all()
        dx, _, _ = nn.linear_backward(y, x, w, wanted=(True, False, False))
        assert torch.isfinite(dx[keep]).all()


def test_without_gradients_nothing_is_kept(nn):
    x, w, b = _operands(50, 45, 40, torch.bfloat16)
    w.requires_grad_()
    with torch.no_grad():
        y = nn.linear(x, w, b, None, "silu", checkpoint="mx8")
    assert not y.requires_grad and torch.equal(y, nn.linear(x, w, b, None, "silu"))


def test_many_rows(nn):
    """More rows than one launch of few rows' kernel takes, x beyond 2^32 bytes."""
    rows = (1 << 27) + 37
    x = torch.zeros(rows, 17, dtype=torch.bfloat16, device="cuda")
    x[-3:] = _normal(70, 3, 17, dtype=torch.bfloat16)
    x[5] = _normal(71, 17, dtype=torch.bfloat16)
    w, b = _normal(72, 3, 17, dtype=torch.bfloat16), _normal(73, 3, dtype=torch.bfloat16)
    y = nn.linear_forward(x, w, b)
    small = nn.linear_forward(x[-3:].contiguous(), w, b)
    assert float((y[-3:].float() - small.float()).abs().max()) <= 2.0 ** -7 * float(small.abs().max())
    assert torch.equal(y[6:-3], b.expand(rows - 9, 3))
    dx, dw, db = nn.linear_backward(y, x, w)
    want = y[-3:].double().t() @ x[-3:].double() + y[5:6].double().t() @ x[5:6].double()
    assert float((dw.double() - want).abs().max()) <= 2.0 ** -7 * float(want.abs().max())
    assert torch.isfinite(dx).all() and dx.shape == x.shape
    del y, dx


def test_residuals_of_another_shape(nn):
    """As many rows in other axes: each gradient has its input's shape."""
    x, w, b = _operands(24, 45, 40, torch.float32)
    r = _normal(74, 24, 40).requires_grad_()
    y = nn.linear(x.view(4, 6, 45), w, b, r, "silu")
    dr, = torch.autograd.grad(y, r, torch.ones_like(y))
    assert y.shape == (4, 6, 40) and dr.shape == (24, 40) and (dr == 1).all()
    n, total = nn.rms_norm(y.detach().requires_grad_(), None, r)
    dr, = torch.autograd.grad(n.sum() + total.sum(), r)
    assert dr.shape == (24, 40)
    dr, = torch.autograd.grad(nn.rms_norm(y.detach(), None, r)[1].sum(), r)
    assert dr.shape == (24, 40) and (dr == 1).all()


def test_two_streams_and_two_graphs_at_once(nn):
    """Calls that overlap have workspaces of their own: streamed weights, parts of sums."""
    sizes = [(17000, 264, 256), (9500, 1000, 200)]
    calls = []
    for i, (rows, inner, outer) in enumerate(sizes):
        x, w, b = _operands(rows, inner, outer, torch.bfloat16, seed=80 + 10 * i)
        dy = _normal(85 + 10 * i, rows, outer, dtype=torch.bfloat16)
        calls.append(lambda x=x, w=w, b=b, dy=dy: (nn.linear_forward(x, w, b, None, "gelu"), *nn.linear_backward(dy, x, w, dy, "silu")))
    want = [[t.clone() for t in c()] for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[], []]
    for _ in range(4):
        for i, (s, c) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(s):
                got[i].append(c())
    torch.cuda.synchronize()
    for g, v in zip(got, want):
        assert all(torch.equal(p, q) for run in g for p, q in zip(run, v))
    graphs, held = [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(c())
        graphs.append(g)
    for _ in range(3):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for h, v in zip(held, want) for p, q in zip(h, v))
        for h in held:
            for t in h:
                t.zero_()
        torch.cuda.synchronize()
