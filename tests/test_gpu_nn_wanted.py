"""Gradients by themselves, and outputs over inputs."""
from __future__ import annotations

import ctypes

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from msplat_amd import _abi  # noqa: E402
from test_gpu_nn import DTYPES, IDS, _ffn_operands, _normal, nn  # noqa: E402, F401


# few rows, split hidden units, resident weights, streamed ones with a tail, no rows
@pytest.mark.parametrize("rows,dim,hidden", [(300, 45, 100), (40, 100, 1100), (20011, 64, 256), (65543, 200, 72),
                                             (0, 45, 100)])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_gated_ffn_gradients_by_themselves(nn, dtype, rows, dim, hidden):  # noqa: F811
    ops, dy = _ffn_operands(rows, dim, hidden, dtype), _normal(30, rows, dim, dtype=dtype)
    dx, *grads = nn.gated_ffn_backward(dy, *ops)
    alone, *none = nn.gated_ffn_backward(dy, *ops, wanted=(True, False))
    assert torch.equal(alone, dx) and none == [None] * 3
    none, *alone = nn.gated_ffn_backward(dy, *ops, wanted=(False, True))
    assert none is None and all(torch.equal(p, q) for p, q in zip(alone, grads))
    assert nn.gated_ffn_backward(dy, *ops, wanted=(False, False)) == (None,) * 4


@pytest.mark.parametrize("rows,dim", [(300, 45), (40000, 64), (5000, 600), (1500, 4099), (0, 45)])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_layer_norm_gradients_by_themselves(nn, dtype, rows, dim):  # noqa: F811
    x, dy, w = _normal(1, rows, dim, dtype=dtype), _normal(2, rows, dim, dtype=dtype), 1 + _normal(3, dim, dtype=dtype)
    _, mean, rstd = nn.layer_norm_forward(x, w)
    whole = nn.layer_norm_backward(dy, x, w, mean, rstd)
    for wanted in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (False,) * 3):
        got = nn.layer_norm_backward(dy, x, w, mean, rstd, wanted)
        assert all((g is None) if not n else torch.equal(g, v) for g, v, n in zip(got, whole, wanted)), wanted


def test_autograd_asks_for_what_is_needed(nn, monkeypatch):  # noqa: F811
    asked = []
    for name in ("layer_norm_backward", "gated_ffn_backward"):
        def spy(*args, plain=getattr(nn, name)):
            out = plain(*args)
            asked.append([g is not None for g in out])
            return out
        monkeypatch.setattr(nn, name, spy)
    x, wg, wu, wd = _ffn_operands(50, 40, 60, torch.float32)
    w, b = 1 + _normal(4, 40), _normal(5, 40)

    def run(*leaves):
        for t in leaves:
            t.requires_grad_()
        asked.clear()
        torch.autograd.grad(nn.gated_ffn(nn.layer_norm(x, w, b), wg, wu, wd).sum(), leaves)
        for t in leaves:
            t.requires_grad_(False)
        return list(asked)

    everything = run(x, w, b, wg, wu, wd)
    assert everything == [[True] * 4, [True] * 3]
    assert run(x) == [[True, False, False, False], [True, False, False]]           # frozen weights
    assert run(wd) == [[False, True, True, True]]                                  # a fixed input
    assert run(b, wg) == [[True] * 4, [False, False, True]]


@pytest.mark.parametrize("dim", [1, 3, 45, 64, 601, 2001, 4099, 8191])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_outputs_over_inputs(nn, dtype, dim):  # noqa: F811
    """y or dx in place, from few rows to several turns of a workgroup, of rows
    that a piece does not divide and that several waves share."""
    lib, number = _abi.load(), nn._DTYPES[dtype]
    for rows in (3, 4200):
        x, dy = _normal(1, rows, dim, dtype=dtype), _normal(2, rows, dim, dtype=dtype)
        w = 1 + _normal(3, dim, dtype=dtype)
        y, mean, rstd = nn.layer_norm_forward(x, w, w)
        dx = nn.layer_norm_backward(dy, x, w, mean, rstd, (True, False, False))[0]
        dropped = nn.dropout_add_forward(x, dy, 0.3, 5, 6)
        a = x.clone()
        args = _abi.LayerNormArgs(nn._stream(x), rows, dim, number, a.data_ptr(), dim, w.data_ptr(), w.data_ptr(), 1e-5,
                                  a.data_ptr(), dim, None, None)
        _abi.check(lib.msplat_hip_layer_norm(ctypes.byref(args)))
        assert torch.equal(a, y)
        for over_x in (True, False):
            a, g = x.clone(), dy.clone()
            args = _abi.LayerNormGradArgs(nn._stream(x), rows, dim, number, g.data_ptr(), dim, a.data_ptr(), dim,
                                          w.data_ptr(), mean.data_ptr(), rstd.data_ptr(), (a if over_x else g).data_ptr(),
                                          dim, None, None, None, 0)
            _abi.check(lib.msplat_hip_layer_norm_backward(ctypes.byref(args)))
            assert torch.equal(a if over_x else g, dx) and torch.equal(g if over_x else a, dy if over_x else x)
            a, g = x.clone(), dy.clone()
            args = _abi.DropoutArgs(nn._stream(x), rows, dim, number, 0.3, 5, 6, a.data_ptr(), dim, g.data_ptr(), dim,
                                    (a if over_x else g).data_ptr(), dim)
            _abi.check(lib.msplat_hip_dropout_add(ctypes.byref(args)))
            assert torch.equal(a if over_x else g, dropped) and torch.equal(g if over_x else a, dy if over_x else x)
