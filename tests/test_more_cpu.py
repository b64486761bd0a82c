"""8-bit rows, the root-mean-square norm and the linear layer without a GPU: the
oracle's formulas against differences and by hand, struct layouts, the refusals of the
C entry points and of msplat_amd.nn."""
from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import more_oracle as orc
import nn_oracle
from msplat_amd import _abi, nn
from test_nn_calls_cpu import _On, context  # noqa: F401
from test_nn_cpu import BF16, F16, F32, _Host, _set, lib  # noqa: F401

MX8 = 3


def test_packing_by_hand():
    x = torch.zeros(4, 33)
    x[0, :4] = torch.tensor([448.0, 17.0, 18.0, 0.001])    # scale 1: steps of 2 from 16 on, of 2^-9 near 0
    x[1, :3] = torch.tensor([449.0, 17.0, -0.3])           # scale 2
    x[2, 32] = 3.0                                         # the second block
    x[3, :2] = torch.tensor([float("inf"), 1.75])
    values, codes = orc.mx8(x)
    assert codes.tolist() == [[127, 1], [128, 1], [1, 120], [119, 1]]
    assert values[0, :4].tolist() == [448.0, 16.0, 18.0, 2.0 ** -9 * 1.0]
    assert values[1, 1].item() in (16.0, 18.0) and abs(values[1, 2].item() + 0.3) <= 0.3 / 16
    assert values[2, 32].item() == 3.0 and torch.isnan(values[3, 0]) and values[3, 1].item() == 1.75


def test_rounding_is_to_the_nearest_of_all_elements():
    """Against the list of the format's 253 numbers."""
    table = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    table = table[torch.isfinite(table)].unique()
    g = torch.Generator().manual_seed(1)
    v = torch.cat((448.0 * (2 * torch.rand(4000, generator=g, dtype=torch.float64) - 1),
                   0.05 * torch.randn(4000, generator=g, dtype=torch.float64)))
    nearest = (v[:, None] - table).abs().amin(1)
    got = orc.e4m3(v)
    assert torch.equal((got - v).abs(), nearest) and torch.isin(got, table).all()


def _double(*shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def test_norm_gradients_match_differences():
    nn_oracle.UT[torch.float64] = (2.0 ** -53, 0.0)
    x, r, w = (_double(*s, seed=i).requires_grad_() for i, s in enumerate(((5, 7), (5, 7), (7,))))

    def norm(x, r, w):
        t = x + r
        return t * (t.square().mean(1, keepdim=True) + 1e-5).rsqrt() * w, t

    assert torch.autograd.gradcheck(norm, (x, r, w), eps=1e-6, atol=1e-7)
    dy, dt = _double(5, 7, seed=4), _double(5, 7, seed=5)
    want = torch.autograd.grad(norm(x, r, w), (x, r, w), (dy, dt))
    t = (x + r).detach()
    rstd = (t.square().mean(1) + 1e-5).rsqrt()
    (dx, dw), _ = orc.rms_norm_grad(dy, t, w.detach(), rstd, dt)
    for a, b in ((dx, want[0]), (dx, want[1]), (dw, want[2])):
        assert (a - b).abs().max() < 1e-12 * (1 + b.abs().max())


@pytest.mark.parametrize("act", [None, "silu", "gelu"])
def test_linear_gradients_match_differences(act):
    nn_oracle.UT[torch.float64] = (2.0 ** -53, 0.0)
    x, w, b, r = (_double(*s, seed=i).requires_grad_() for i, s in enumerate(((5, 7), (6, 7), (6,), (5, 6))))

    def linear(x, w, b, r):
        z = x @ w.t() + b
        return r + (z if act is None else nn_oracle.activation(z, act)[0])

    assert torch.autograd.gradcheck(linear, (x, w, b, r), eps=1e-6, atol=1e-7)
    dy = _double(5, 6, seed=4)
    want = torch.autograd.grad(linear(x, w, b, r), (x, w, b, r), dy)
    z = (x @ w.t() + b).detach()
    got, _ = orc.linear_grad(dy, x.detach(), w.detach(), z, act, torch.float64)
    for a, v in zip((*got, dy), want):
        assert (a - v).abs().max() < 1e-12 * (1 + v.abs().max())


STRUCTS = {"MsplatMx8Args": _abi.Mx8Args, "MsplatRmsNormArgs": _abi.RmsNormArgs,
           "MsplatRmsNormGradArgs": _abi.RmsNormGradArgs, "MsplatLinearArgs": _abi.LinearArgs,
           "MsplatLinearGradArgs": _abi.LinearGradArgs}


def test_struct_layouts_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if not cc:
        pytest.skip("no host C compiler")
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "msplat_hip.h")
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {"]
    for name, py in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in py._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.check_call([cc, "-std=c99", "-o", str(exe), str(src)])
    got = dict(line.rsplit(" ", 1) for line in subprocess.check_output([str(exe)], text=True).splitlines())
    for name, py in STRUCTS.items():
        assert int(got[name]) == ctypes.sizeof(py)
        for f in py._fields_:
            assert int(got[f"{name}.{f[0]}"]) == getattr(py, f[0]).offset, (name, f[0])


def _mx8(**kw):
    h = _Host()
    return h, _set(_abi.Mx8Args(None, 2, 4, F32, h.at, 4, h.at, h.at), kw)


def _rms(**kw):
    h = _Host()
    return h, _set(_abi.RmsNormArgs(None, 2, 4, F32, h.at, 4, h.at, 4, h.at, 1e-5, h.at, 4, None, h.at + 64, 4, h.at), kw)


def _rms_grad(**kw):
    h = _Host()
    a = _abi.RmsNormGradArgs(None, 2, 4, F32, h.at, 4, h.at, 4, h.at, 4, None, h.at, h.at, h.at, 4, h.at, h.at, 1 << 20)
    return h, _set(a, kw)


def _linear(**kw):
    h = _Host()
    a = _abi.LinearArgs(None, 2, 4, 8, F32, F32, 0, h.at, 4, None, h.at, 4, None, h.at, h.at, 8, h.at, 8, h.at + 64, 8, h.at,
                        1 << 20)
    return h, _set(a, kw)


def _linear_grad(**kw):
    h = _Host()
    a = _abi.LinearGradArgs(None, 2, 4, 8, F32, F32, 0, h.at, 8, h.at, 4, None, h.at, 4, h.at, 8, None, h.at, 4, h.at, h.at,
                            h.at, 1 << 20)
    return h, _set(a, kw)


CALLS = {"msplat_hip_mx8_pack": _mx8, "msplat_hip_mx8_unpack": _mx8, "msplat_hip_rms_norm": _rms,
         "msplat_hip_rms_norm_backward": _rms_grad, "msplat_hip_linear": _linear,
         "msplat_hip_linear_backward": _linear_grad}
COMMON = [(dict(rows=-1), b"rows"), (dict(rows=1 << 31), b"rows"), (dict(dtype=7), b"dtype")]
DIM = [(dict(dim=0), b"dim"), (dict(dim=-4), b"dim")]
SIZES = [(dict(inner=0), b"dim"), (dict(inner=65537, x_stride=65537), b"dim"), (dict(outer=0), b"outer"),
         (dict(outer=65537), b"outer"), (dict(activation=3), b"activation"), (dict(activation=-1), b"activation"),
         (dict(y_dtype=3), b"y_dtype"), (dict(x=None), b"x is null"), (dict(x_stride=3), b"stride"),
         (dict(weight=None), b"weight is null"), (dict(weight_stride=3), b"stride")]
PACKED = [(dict(matrix=None), b"null"), (dict(data=None), b"null"), (dict(scales=None), b"null"), (dict(stride=3), b"stride"),
          (dict(dim=(1 << 30) + 1, stride=1 << 31), b"dim")]
OWN = {
    "msplat_hip_mx8_pack": DIM + PACKED, "msplat_hip_mx8_unpack": DIM + PACKED,
    "msplat_hip_rms_norm": DIM + [(dict(dim=8193, x_stride=8193), b"dim"), (dict(x=None), b"x is null"),
                                  (dict(y=None), b"y is null"), (dict(y_stride=1), b"stride"), (dict(eps=-1.0), b"eps"),
                                  (dict(eps=float("nan")), b"eps"), (dict(residual_stride=1), b"stride"),
                                  (dict(total_stride=1), b"stride")],
    "msplat_hip_rms_norm_backward": DIM + [(dict(dy=None), b"dy is null"), (dict(total=None), b"total is null"),
                                           (dict(rstd=None), b"rstd"), (dict(dtotal_stride=3), b"stride"),
                                           (dict(dx_stride=3), b"stride"), (dict(workspace=None), b"workspace"),
                                           (dict(workspace_bytes=8), b"workspace")],
    "msplat_hip_linear": SIZES + [(dict(y=None), b"y is null"), (dict(y_stride=7), b"stride"),
                                  (dict(residual_stride=7), b"stride"), (dict(z_stride=7), b"stride")],
    "msplat_hip_linear_backward": SIZES + [(dict(dy=None), b"dy is null"), (dict(dy_stride=7), b"stride"),
                                           (dict(z=None), b"z is null"), (dict(z_stride=7), b"stride"),
                                           (dict(dx_stride=3), b"stride"), (dict(workspace=None), b"workspace"),
                                           (dict(workspace_bytes=16), b"workspace"), (dict(dtype=MX8), b"dtype")],
}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_refusals(lib, name):  # noqa: F811
    fn = getattr(lib, name)
    assert fn(None) == -1
    for kw, word in COMMON + OWN[name]:
        _, a = CALLS[name](**kw)
        assert fn(ctypes.byref(a)) == -1, kw
        assert word in lib.msplat_hip_last_error(), (kw, lib.msplat_hip_last_error())


@pytest.mark.parametrize("name,fields", [
    ("msplat_hip_mx8_pack", ("matrix", "data", "scales")), ("msplat_hip_mx8_unpack", ("matrix", "data", "scales")),
    ("msplat_hip_rms_norm", ("x", "residual", "weight", "y", "total", "rstd")),
    ("msplat_hip_rms_norm_backward", ("dy", "dtotal", "total", "weight", "rstd", "dx", "dweight", "workspace")),
    ("msplat_hip_linear", ("x", "weight", "bias", "residual", "y", "z")),
    ("msplat_hip_linear_backward", ("dy", "x", "weight", "z", "dx", "dweight", "dbias", "workspace"))])
def test_misaligned_operands_are_refused(lib, name, fields):  # noqa: F811
    for field in fields:
        h, a = CALLS[name]()
        setattr(a, field, h.at + 2)
        assert getattr(lib, name)(ctypes.byref(a)) == -1, field
        assert b"align" in lib.msplat_hip_last_error(), field


def test_8_bit_operands_are_checked(lib):  # noqa: F811
    """Data and scales are both there, on 16-byte boundaries, and go with the type that says so."""
    h, a = _rms()
    a.y_scales = h.at + 4
    assert lib.msplat_hip_rms_norm(ctypes.byref(a)) == -1 and b"16-byte" in lib.msplat_hip_last_error()
    h, a = _rms_grad()
    a.total_scales = h.at + 8
    assert lib.msplat_hip_rms_norm_backward(ctypes.byref(a)) == -1 and b"16-byte" in lib.msplat_hip_last_error()
    for field in ("x_scales", "z_scales"):
        h, a = _linear_grad()
        setattr(a, field, h.at + 4)
        assert lib.msplat_hip_linear_backward(ctypes.byref(a)) == -1 and b"16-byte" in lib.msplat_hip_last_error()
    h, a = _linear(x_scales=16)
    assert lib.msplat_hip_linear(ctypes.byref(a)) == -1 and b"scales" in lib.msplat_hip_last_error()
    h, a = _linear(dtype=MX8)
    assert lib.msplat_hip_linear(ctypes.byref(a)) == -1 and b"x is null" in lib.msplat_hip_last_error()
    a.x_scales = h.at
    assert lib.msplat_hip_linear(ctypes.byref(a)) == -1 and b"weight is null" in lib.msplat_hip_last_error()
    a.weight_scales = h.at
    assert lib.msplat_hip_linear(ctypes.byref(a)) == -1 and b"z is not kept" in lib.msplat_hip_last_error()


def test_results_in_one_place_are_refused(lib):  # noqa: F811
    h, a = _rms()
    a.total = a.y
    assert lib.msplat_hip_rms_norm(ctypes.byref(a)) == -1 and b"same matrix" in lib.msplat_hip_last_error()
    h, a = _linear()
    a.z = a.y
    assert lib.msplat_hip_linear(ctypes.byref(a)) == -1 and b"same matrix" in lib.msplat_hip_last_error()


@pytest.mark.parametrize("name", sorted(CALLS))
def test_valid_arguments_reach_the_context_check(lib, name):  # noqa: F811
    from msplat_amd import device
    if device._initialised:
        pytest.skip("a context already exists in this process")
    _, a = CALLS[name]()
    assert getattr(lib, name)(ctypes.byref(a)) == -3


def test_workspace_sizes(lib):  # noqa: F811
    rms, fwd, bwd = (lib.msplat_hip_rms_norm_backward_workspace, lib.msplat_hip_linear_workspace,
                     lib.msplat_hip_linear_backward_workspace)
    assert rms(10, 8193, F32) == -1 and rms(-1, 8, F32) == -1 and rms(1, 8, 5) == -1
    assert 0 < rms(1, 8192, F32) <= rms((1 << 31) - 1, 8192, F32) < 1 << 26
    assert fwd(1, 0, 8, F32) == fwd(1, 8, 65537, F32) == fwd(1, 8, 8, 4) == -1
    assert bwd(1, 8, 8, MX8, F32, 0) == bwd(1, 8, 8, F32, 5, 0) == bwd(1, 8, 8, F32, F32, 4) == -1
    for dtype in (F32, F16, BF16):
        assert bwd(0, 8, 8, dtype, dtype, 0) == 0
        for inner, outer in ((1, 1), (64, 256), (1000, 200), (65536, 65536)):
            assert fwd(1, inner, outer, MX8) >= 0
            # weights of at most twice their size, and of a column block and four of the contraction
            for rows in (1, 100_000, (1 << 31) - 1):
                assert 0 <= fwd(rows, inner, outer, dtype) <= 2 * 4 * (inner + 128) * (outer + 64) * 2
                assert 0 < bwd(rows, inner, outer, dtype, dtype, 2) < 1 << 42


def test_python_refusals():
    x = torch.zeros(4, 8)
    m = nn.Mx8(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 8, torch.float32)
    assert m.shape == (4, 8) and m.rows == 4
    for call in (lambda: nn.mx8_pack(x), lambda: nn.mx8_unpack(m), lambda: nn.rms_norm_forward(x),
                 lambda: nn.rms_norm_backward(x, x, None, torch.zeros(4)), lambda: nn.linear_forward(x, x),
                 lambda: nn.linear_forward(m, m), lambda: nn.linear_backward(x, x, x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call, word in ((lambda: nn.linear_forward(x, x, activation="relu"), "activation"),
                       (lambda: nn.linear_forward(m, x), "both Mx8"), (lambda: nn.linear_forward(x, m), "both Mx8"),
                       (lambda: nn.linear(x, x, checkpoint="int4"), "checkpoint"),
                       (lambda: nn.linear(m, m), "no gradients"), (lambda: nn.linear(x, m), "no gradients"),
                       (lambda: nn.rms_norm(x, checkpoint="fp8"), "checkpoint"),
                       (lambda: nn.gated_ffn(x, x, x, x, checkpoint="fp8"), "checkpoint")):
        with pytest.raises(ValueError, match=word):
            call()


def test_an_mx8_is_checked():
    d, s = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8)
    assert nn.Mx8(d, s, 33, torch.float16).shape == (4, 33)
    assert nn.Mx8(d.view(torch.float8_e4m3fn), s, 64, torch.bfloat16).dtype is torch.bfloat16
    for args in ((d, s, 32, torch.float32), (d, s, 65, torch.float32), (d, s, 0, torch.float32),
                 (d, s[:3], 64, torch.float32), (d, torch.zeros(4, 2, dtype=torch.uint8), 64, torch.float32),
                 (d.float(), s, 64, torch.float32), (d, s.float(), 64, torch.float32), (d, s, 64, torch.int8)):
        with pytest.raises(ValueError):
            nn.Mx8(*args)
    # rows of a larger buffer that start off the boundary are moved
    off = torch.zeros(4 * 64 + 8, dtype=torch.uint8)[8:].view(4, 64)
    assert nn.Mx8(off, s, 64, torch.float32).data.data_ptr() % 16 == 0
    # a slice of rows is a matrix by itself
    assert nn.Mx8(d[1:3], s[1:3], 64, torch.float32).rows == 2


def test_another_gpus_tensors_are_refused(context):  # noqa: F811
    far = _On(1)
    for call in (lambda: nn.mx8_pack(far), lambda: nn.rms_norm_forward(far), lambda: nn.rms_norm_backward(far, far, None, None),
                 lambda: nn.linear_forward(far, far), lambda: nn.linear_backward(far, far, far)):
        with pytest.raises(ValueError, match="cuda:1"):
            call()
