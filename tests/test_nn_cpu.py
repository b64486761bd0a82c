"""Learned-head operators without a GPU: the oracle's formulas against
differences and published values, and the refusals of the C entry points."""
from __future__ import annotations

import ctypes
import os

import numpy as np
import pytest
import torch

import nn_oracle as orc
from msplat_amd import _abi

F32, F16, BF16 = 0, 1, 2


def test_philox_matches_the_published_vectors():
    """Known answers of Philox 4x32 with ten rounds, as its authors publish
    them; the mask's seven rounds are the same code."""
    zero = [int(v) for v in orc.philox((0, 0, 0, 0), (0, 0), 10)]
    assert zero == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    f = 0xFFFFFFFF
    ones = [int(v) for v in orc.philox((f, f, f, f), (f, f), 10)]
    assert ones == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_mask_keeps_its_share_in_every_column():
    """20000 rows: a column's share of kept elements is within five standard
    deviations (0.0153 at p = 0.25) of 1 - p."""
    keep = orc.keep_mask(20000, 13, 0.25, 0x123456789ABCDEF, 7).double()
    assert (keep.mean(0) - 0.75).abs().max() < 5 * (0.25 * 0.75 / 20000) ** 0.5
    other = orc.keep_mask(20000, 13, 0.25, 0x123456789ABCDEF, 8).double()
    assert 0.6 < (keep == other).double().mean() < 0.65   # 0.75^2 + 0.25^2


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_ffn_gradient_formulas_match_differences(act):
    g = torch.Generator().manual_seed(3)
    t = [torch.randn(s, generator=g, dtype=torch.float64).requires_grad_()
         for s in ((5, 7), (6, 7), (6, 7), (7, 6))]
    assert torch.autograd.gradcheck(lambda *a: orc.gated_ffn(*a, act), t, eps=1e-6, atol=1e-7)
    dy = torch.randn(5, 7, generator=g, dtype=torch.float64)
    want = torch.autograd.grad(orc.gated_ffn(*t, act), t, dy)
    x, wg, wu, wd = (v.detach() for v in t)
    # the bounds' types are looked up by the inputs' own
    orc.UT[torch.float64] = (2.0 ** -53, 0.0)
    got, _ = orc.gated_ffn_grad_bounds(dy, x, wg, wu, wd, act)
    for a, b in zip(got, want):
        assert (a - b).abs().max() < 1e-12 * (1 + b.abs().max())


def test_norm_gradient_formulas_match_differences():
    g = torch.Generator().manual_seed(4)
    x = torch.randn(5, 7, generator=g, dtype=torch.float64).requires_grad_()
    w = torch.randn(7, generator=g, dtype=torch.float64).requires_grad_()
    b = torch.randn(7, generator=g, dtype=torch.float64).requires_grad_()

    def norm(x, w, b):
        d = x - x.mean(1, keepdim=True)
        return d * (d.square().mean(1, keepdim=True) + 1e-5).rsqrt() * w + b

    assert torch.autograd.gradcheck(norm, (x, w, b), eps=1e-6, atol=1e-7)
    dy = torch.randn(5, 7, generator=g, dtype=torch.float64)
    want = torch.autograd.grad(norm(x, w, b), (x, w, b), dy)
    orc.UT[torch.float64] = (2.0 ** -53, 0.0)
    (_, mean, rstd), _ = orc.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5)
    got, _ = orc.layer_norm_grad(dy, x.detach(), w.detach(), mean, rstd)
    for p, q in zip(got, want):
        assert (p - q).abs().max() < 1e-12 * (1 + q.abs().max())


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_abi.LIB_PATH):
        pytest.skip("libmsplat_hip.so not built")
    return _abi.load()


class _Host:
    """Host memory that stands in for operands: the refusals come before anything reads them."""

    def __init__(self):
        self.buf = (ctypes.c_double * 66)()
        self.at = (ctypes.addressof(self.buf) + 15) // 16 * 16


def _norm(**kw):
    h = _Host()
    a = _abi.LayerNormArgs(None, 2, 4, F32, h.at, 4, None, None, 1e-5, h.at, 4, None, None)
    return h, _set(a, kw)


def _norm_grad(**kw):
    h = _Host()
    a = _abi.LayerNormGradArgs(None, 2, 4, F32, h.at, 4, h.at, 4, None, h.at, h.at, h.at, 4, h.at, h.at, h.at, 1 << 20)
    return h, _set(a, kw)


def _ffn(**kw):
    h = _Host()
    a = _abi.GatedFfnArgs(None, 2, 4, 8, F32, 0, h.at, 4, h.at, 4, h.at, 4, h.at, 8, h.at, 4, h.at, 1 << 30)
    return h, _set(a, kw)


def _ffn_grad(**kw):
    h = _Host()
    a = _abi.GatedFfnGradArgs(None, 2, 4, 8, F32, 0, h.at, 4, h.at, 4, h.at, 4, h.at, 4, h.at, 8, h.at, 4, h.at, h.at,
                              h.at, h.at, 1 << 30)
    return h, _set(a, kw)


def _drop(**kw):
    h = _Host()
    a = _abi.DropoutArgs(None, 2, 4, F32, 0.5, 1, 2, h.at, 4, h.at, 4, h.at, 4)
    return h, _set(a, kw)


def _set(a, kw):
    for k, v in kw.items():
        setattr(a, k, v)
    return a


CALLS = {"msplat_hip_layer_norm": _norm, "msplat_hip_layer_norm_backward": _norm_grad,
         "msplat_hip_gated_ffn": _ffn, "msplat_hip_gated_ffn_backward": _ffn_grad, "msplat_hip_dropout_add": _drop}
COMMON = [(dict(rows=-1), b"rows"), (dict(rows=1 << 31), b"rows"), (dict(dim=0), b"dim"), (dict(dtype=3), b"dtype"),
          (dict(x=None), b"x is null"), (dict(x_stride=3), b"stride")]
OWN = {
    "msplat_hip_layer_norm": [(dict(dim=8193, x_stride=8193, y_stride=8193), b"dim"), (dict(y=None), b"y is null"),
                              (dict(y_stride=1), b"stride"), (dict(eps=-1.0), b"eps"),
                              (dict(eps=float("nan")), b"eps")],
    "msplat_hip_layer_norm_backward": [(dict(dy=None), b"dy is null"), (dict(mean=None), b"mean"),
                                       (dict(rstd=None), b"rstd"), (dict(workspace=None), b"workspace"),
                                       (dict(workspace_bytes=8), b"workspace"), (dict(dx_stride=2), b"stride")],
    "msplat_hip_gated_ffn": [(dict(dim=257), b"dim"), (dict(hidden=0), b"hidden"), (dict(hidden=65537), b"hidden"),
                             (dict(activation=2), b"activation"), (dict(w_gate=None), b"w_gate"),
                             (dict(w_up=None), b"w_up"), (dict(w_down=None), b"w_down"),
                             (dict(down_stride=7), b"stride"), (dict(workspace=None), b"workspace"),
                             (dict(workspace_bytes=16), b"workspace"), (dict(y=None), b"y is null")],
    "msplat_hip_gated_ffn_backward": [(dict(dim=257), b"dim"), (dict(hidden=0), b"hidden"),
                                      (dict(activation=-1), b"activation"), (dict(dy=None), b"dy is null"),
                                      (dict(dw_up=None), b"together"), (dict(workspace_bytes=16), b"workspace"),
                                      (dict(dx_stride=1), b"stride")],
    "msplat_hip_dropout_add": [(dict(p=-0.1), b"p "), (dict(p=1.5), b"p "), (dict(p=float("nan")), b"p "),
                               (dict(residual_stride=1), b"stride"), (dict(y=None), b"y is null")],
}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_refusals(lib, name):
    fn = getattr(lib, name)
    assert fn(None) == -1
    for kw, word in COMMON + OWN[name]:
        _, a = CALLS[name](**kw)
        assert fn(ctypes.byref(a)) == -1, kw
        assert word in lib.msplat_hip_last_error(), (kw, lib.msplat_hip_last_error())


@pytest.mark.parametrize("name", sorted(CALLS))
def test_misaligned_matrix_is_refused(lib, name):
    h, a = CALLS[name]()
    a.x = h.at + 2
    assert getattr(lib, name)(ctypes.byref(a)) == -1
    assert b"aligned" in lib.msplat_hip_last_error()


def test_misaligned_vectors_are_refused(lib):
    for name, fields in (("msplat_hip_layer_norm", ("weight", "bias", "mean", "rstd")),
                         ("msplat_hip_layer_norm_backward", ("weight", "mean", "rstd", "dweight", "dbias")),
                         ("msplat_hip_gated_ffn_backward", ("dw_gate", "dw_up", "dw_down"))):
        for field in fields:
            h, a = CALLS[name]()
            setattr(a, field, h.at + 2)
            assert getattr(lib, name)(ctypes.byref(a)) == -1, (name, field)
            assert field.encode() in lib.msplat_hip_last_error()


def test_misaligned_workspace_is_refused(lib):
    for name in ("msplat_hip_gated_ffn", "msplat_hip_gated_ffn_backward"):
        h, a = CALLS[name]()
        a.workspace = h.at + 8
        assert getattr(lib, name)(ctypes.byref(a)) == -1
        assert b"16-byte" in lib.msplat_hip_last_error()


@pytest.mark.parametrize("name", sorted(CALLS))
def test_valid_arguments_reach_the_context_check(lib, name):
    from msplat_amd import device
    if device._initialised:
        pytest.skip("a context already exists in this process")
    _, a = CALLS[name]()
    assert getattr(lib, name)(ctypes.byref(a)) == -3


def test_workspace_sizes(lib):
    ffn, ffn_b = lib.msplat_hip_gated_ffn_workspace, lib.msplat_hip_gated_ffn_backward_workspace
    for f in (ffn, ffn_b):
        assert f(100, 257, 8, F32) == -1 and f(100, 8, 0, F32) == -1 and f(-1, 8, 8, F32) == -1
        assert f(100, 8, 8, 9) == -1
        for dtype in (F32, F16, BF16):
            for dim, hidden in ((1, 1), (64, 256), (256, 65536)):
                assert 0 < f(0, dim, hidden, dtype) <= f(1 << 20, dim, hidden, dtype) < 1 << 31
    norm = lib.msplat_hip_layer_norm_backward_workspace
    assert norm(10, 8193, F32) == -1
    assert 0 < norm(1, 8192, F32) <= norm((1 << 31) - 1, 8192, F32) < 1 << 27


def test_python_refusals():
    from msplat_amd import nn
    x = torch.zeros(4, 8)
    for call in (lambda: nn.layer_norm_forward(x), lambda: nn.dropout_add_forward(x, None, 0.5, 1, 2),
                 lambda: nn.gated_ffn_forward(x, torch.zeros(4, 8), torch.zeros(4, 8), torch.zeros(8, 4))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
