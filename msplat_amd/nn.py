"""Operators of a learned head, trained next to a scene.

Layer norm, root-mean-square norm with the residual's addition, a linear layer
with bias, activation and residual, a gated feed-forward block and dropout added to
a residual, over the features of gaussians or pixels: CUDA tensors [..., dim] of
float32, float16 or bfloat16 (one type a call), with any stride between rows, on the
GPU of the library's context (the first call's, if none has made one yet).  Each
runs hand-written kernels of libmsplat_hip.so on PyTorch's current stream, sums
in fp32, and has

  layer_norm, rms_norm, linear, gated_ffn, dropout_add   differentiable by autograd
  *_forward, *_backward                                  the two passes by themselves

Rows in 8 bits (Mx8, mx8_pack, mx8_unpack) are what the backward passes of rms_norm
and linear take instead of their forward's inputs, rms_norm writes and linear
multiplies; checkpoint="mx8" keeps a training step's activations so where they are
smaller that way (rows of few columns are not).

None of them waits for the GPU or keeps anything between calls, so they may
be captured into a graph.  A replay repeats a call's arguments: where each is to
drop other elements, dropout takes its offset as a tensor.  As with PyTorch's own
functions, no graph of autograd's from outside the capture may be alive over the same
leaves while a backward pass is captured.
"""
from __future__ import annotations

import ctypes
from operator import index   # numpy's integers overflow in & where Python's do not
from typing import Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _abi, device

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ACTIVATIONS = {"silu": 0, "gelu": 1}


def _library(t):
    gpu = t.get_device()
    if gpu < 0:
        raise ValueError("the operators take CUDA tensors")
    return device.init_for(gpu)


_DEFAULT_STREAM = 0xFFFFFFFFFFFFFFFF   # MSPLAT_DEFAULT_STREAM


def _stream(t) -> int:
    """PyTorch's current stream.  The library's own stream would do for the
    default one, but each change between the two costs the GPU some 10 us."""
    # the stream object of torch.cuda.current_stream costs 2 us a call
    return torch._C._cuda_getCurrentRawStream(t.device.index) or _DEFAULT_STREAM


def _plain(t) -> bool:
    """Whether a matrix has adjacent columns and rows that do not overlap (an
    expanded gradient's do)."""
    rows, cols = t.shape
    return (t.stride(1) == 1 or cols == 1) and (t.stride(0) >= cols or rows <= 1)


def _tensor(name, t):
    if type(t) is Mx8:
        raise ValueError(f"{name} is an Mx8 where a tensor is taken")


def _rows(name, t, dim, like):
    """t as a [rows, dim] matrix with adjacent columns."""
    _tensor(name, t)
    if t.dim() == 2 and t.is_contiguous() and t.shape[1] == dim and t.dtype is like.dtype and \
            t.get_device() == like.get_device():
        return t
    if t.dtype is not like.dtype or t.device != like.device:
        raise ValueError(f"{name} is {t.dtype} on {t.device}, not {like.dtype} on {like.device}")
    if t.dim() < 1 or t.shape[-1] != dim:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not [..., {dim}]")
    if t.dim() != 2:
        t = t.reshape(-1, dim)
    return t if _plain(t) else t.contiguous()


def _matrix(name, t, shape, like):
    _tensor(name, t)
    if t.shape == shape and t.is_contiguous() and t.dtype is like.dtype and t.get_device() == like.get_device():
        return t
    if t.dtype is not like.dtype or t.device != like.device:
        raise ValueError(f"{name} is {t.dtype} on {t.device}, not {like.dtype} on {like.device}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {shape}")
    return t if (t.stride(0) == 1 if len(shape) == 1 else _plain(t)) else t.contiguous()


def _dtype(t) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise ValueError(f"{t.dtype} is none of float32, float16, bfloat16") from None


def _feature_rows(name, x):
    _tensor(name, x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} has shape {tuple(x.shape)}, not [..., dim]")
    return x if x.dim() == 2 and x.is_contiguous() else _rows(name, x, x.shape[-1], x)


def _same_rows(name, t, x2):
    t2 = _rows(name, t, x2.shape[1], x2)
    if t2.shape[0] != x2.shape[0]:
        raise ValueError(f"{name} has {t2.shape[0]} rows, not {x2.shape[0]}")
    return t2


def _workspace(nbytes, like):
    if nbytes < 0:
        raise _abi.MsplatError(f"msplat_hip error: {_abi.load().msplat_hip_last_error().decode()}")
    return like.new_empty(-(-nbytes // like.element_size()))


def _ptr(t):
    return None if t is None else t.data_ptr()


def layer_norm_forward(x, weight=None, bias=None, eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): y = (x - mean) rstd weight + bias over the last axis, of
    x's type; mean and rstd, one float32 a row, are what the backward takes."""
    lib, dtype = _library(x), _dtype(x)
    x2 = _feature_rows("x", x)
    rows, dim = x2.shape
    w = None if weight is None else _matrix("weight", weight, (dim,), x)
    b = None if bias is None else _matrix("bias", bias, (dim,), x)
    y = x.new_empty(x.shape)
    mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
    rstd = mean.new_empty(mean.shape)
    a = _abi.LayerNormArgs(_stream(x), rows, dim, dtype, x2.data_ptr(), x2.stride(0), _ptr(w), _ptr(b), eps,
                           y.data_ptr(), dim, mean.data_ptr(), rstd.data_ptr())
    _abi.check(lib.msplat_hip_layer_norm(ctypes.byref(a)))
    return y, mean, rstd


def layer_norm_backward(dy, x, weight, mean, rstd, wanted=(True, True, True)):
    """(dx, dweight, dbias) from the gradient of y and the forward's x, mean
    and rstd; dweight and dbias have x's type, also where weight is None.
    Those not wanted are None and not computed."""
    lib, dtype = _library(x), _dtype(x)
    x2 = _feature_rows("x", x)
    rows, dim = x2.shape
    dy2 = _same_rows("dy", dy, x2)
    w = None if weight is None else _matrix("weight", weight, (dim,), x)
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.dtype is not torch.float32 or t.numel() != rows or t.device != x.device:
            raise ValueError(f"{name} must hold one float32 a row on {x.device}")
    mean, rstd = mean.contiguous(), rstd.contiguous()
    dx = x.new_empty(x.shape) if wanted[0] else None
    dweight = x.new_empty(dim) if wanted[1] else None
    dbias = x.new_empty(dim) if wanted[2] else None
    ws = _workspace(lib.msplat_hip_layer_norm_backward_workspace(rows, dim, dtype), x)
    a = _abi.LayerNormGradArgs(_stream(x), rows, dim, dtype, dy2.data_ptr(), dy2.stride(0), x2.data_ptr(),
                               x2.stride(0), _ptr(w), mean.data_ptr(), rstd.data_ptr(), _ptr(dx), dim,
                               _ptr(dweight), _ptr(dbias), ws.data_ptr(), ws.nbytes)
    _abi.check(lib.msplat_hip_layer_norm_backward(ctypes.byref(a)))
    return dx, dweight, dbias


def _ffn_operands(x, w_gate, w_up, w_down, activation):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation {activation!r} is none of {sorted(_ACTIVATIONS)}")
    x2 = _feature_rows("x", x)
    dim = x2.shape[1]
    if w_gate.dim() != 2:
        raise ValueError(f"w_gate has shape {tuple(w_gate.shape)}, not (hidden, {dim})")
    hidden = w_gate.shape[0]
    return (x2, hidden, _matrix("w_gate", w_gate, (hidden, dim), x), _matrix("w_up", w_up, (hidden, dim), x),
            _matrix("w_down", w_down, (dim, hidden), x))


def gated_ffn_forward(x, w_gate, w_up, w_down, activation: str = "silu"):
    """(a(x w_gate^T) * (x w_up^T)) w_down^T with a = SiLU or GELU (tanh form);
    w_gate and w_up [hidden, dim], w_down [dim, hidden], dim at most 256.  In
    16-bit types the hidden units are rounded to the type (float16: infinite
    beyond 65504)."""
    lib, dtype = _library(x), _dtype(x)
    x2, hidden, wg, wu, wd = _ffn_operands(x, w_gate, w_up, w_down, activation)
    rows, dim = x2.shape
    y = x.new_empty(x.shape)
    ws = _workspace(lib.msplat_hip_gated_ffn_workspace(rows, dim, hidden, dtype), x)
    a = _abi.GatedFfnArgs(_stream(x), rows, dim, hidden, dtype, _ACTIVATIONS[activation], x2.data_ptr(),
                          x2.stride(0), wg.data_ptr(), wg.stride(0), wu.data_ptr(), wu.stride(0), wd.data_ptr(),
                          wd.stride(0), y.data_ptr(), dim, ws.data_ptr(), ws.nbytes)
    _abi.check(lib.msplat_hip_gated_ffn(ctypes.byref(a)))
    return y


def gated_ffn_backward(dy, x, w_gate, w_up, w_down, activation: str = "silu", wanted=(True, True)):
    """(dx, dw_gate, dw_up, dw_down) from the gradient of y, x and the weights.
    wanted: dx, and the three weights' together; those that are not are None and
    not computed.  In 16-bit types the hidden units' gradients are rounded to the
    type (float16: fewer bits below 6e-5, 0 below 3e-8)."""
    lib, dtype = _library(x), _dtype(x)
    x2, hidden, wg, wu, wd = _ffn_operands(x, w_gate, w_up, w_down, activation)
    rows, dim = x2.shape
    dy2 = _same_rows("dy", dy, x2)
    dx = x.new_empty(x.shape) if wanted[0] else None
    shapes = (hidden, dim), (hidden, dim), (dim, hidden)
    grads = [x.new_empty(s) if wanted[1] else None for s in shapes]
    ws = _workspace(lib.msplat_hip_gated_ffn_backward_workspace(rows, dim, hidden, dtype), x)
    a = _abi.GatedFfnGradArgs(_stream(x), rows, dim, hidden, dtype, _ACTIVATIONS[activation], dy2.data_ptr(),
                              dy2.stride(0), x2.data_ptr(), x2.stride(0), wg.data_ptr(), wg.stride(0),
                              wu.data_ptr(), wu.stride(0), wd.data_ptr(), wd.stride(0), _ptr(dx), dim,
                              _ptr(grads[0]), _ptr(grads[1]), _ptr(grads[2]), ws.data_ptr(), ws.nbytes)
    _abi.check(lib.msplat_hip_gated_ffn_backward(ctypes.byref(a)))
    return (dx, *grads)


def _dropout(x, residual, p, seed, offset):
    lib, dtype = _library(x), _dtype(x)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p = {p} is outside [0, 1]")
    x2 = _feature_rows("x", x)
    rows, dim = x2.shape
    r2 = None if residual is None else _same_rows("residual", residual, x2)
    y = x.new_empty(x.shape)
    at = offset if torch.is_tensor(offset) else None
    if at is not None and (at.dtype is not torch.int64 or at.numel() != 1 or at.device != x.device):
        raise ValueError(f"offset must be a number or one int64 on {x.device}")
    number = 0 if at is not None else index(offset) & 0xFFFFFFFFFFFFFFFF
    a = _abi.DropoutArgs(_stream(x), rows, dim, dtype, p, index(seed) & 0xFFFFFFFFFFFFFFFF, number, x2.data_ptr(),
                         x2.stride(0), _ptr(r2), 0 if r2 is None else r2.stride(0), y.data_ptr(), dim)
    if at is None:
        _abi.check(lib.msplat_hip_dropout_add(ctypes.byref(a)))
    else:
        _abi.check(lib.msplat_hip_dropout_add_at(ctypes.byref(a), at.data_ptr()))
    return y


def dropout_add_forward(x, residual, p: float, seed: int, offset):
    """residual + keep * x / (1 - p); residual None for none.  The mask is
    a function of seed, offset, row and column (the first axes count as one)
    and is never stored; give each layer its seed and each step its offset: a
    number, or a tensor of one int64 on x's GPU that is read when the kernel
    runs, so that replays of a captured step may differ in it."""
    return _dropout(x, residual, p, seed, offset)


def dropout_add_backward(dy, p: float, seed: int, offset):
    """The gradient of dropout_add's x; the residual's is dy itself."""
    return _dropout(dy, None, p, seed, offset)


class Mx8:
    """Numbers [..., dim] in 8 bits, as mx8_pack and rms_norm_forward write them:
    the OCP microscaling format MXFP8.  data: e4m3 bytes [..., 32 ceil(dim / 32)],
    zeros from dim on; scales: a byte for each 32 adjacent columns, 127 + the
    exponent of a power of two, [..., 4 ceil(dim / 128)]; both contiguous.  dtype:
    the type that they stand in for."""

    __slots__ = ("data", "scales", "dim", "dtype")

    def __init__(self, data, scales, dim: int, dtype):
        dim = index(dim)
        if dtype not in _DTYPES:
            raise ValueError(f"{dtype} is none of float32, float16, bfloat16")
        if data.dtype not in (torch.uint8, torch.float8_e4m3fn) or scales.dtype is not torch.uint8:
            raise ValueError(f"data is {data.dtype} and scales {scales.dtype}, not float8_e4m3fn (or uint8) and uint8")
        if dim < 1 or data.dim() < 1 or scales.dim() < 1 or scales.shape != (*data.shape[:-1], 4 * -(-dim // 128)) or \
                data.shape[-1] != 32 * -(-dim // 32):
            raise ValueError(f"data of shape {tuple(data.shape)} and scales of {tuple(scales.shape)} do not hold "
                             f"[..., {dim}]")
        if data.device != scales.device:
            raise ValueError(f"data is on {data.device}, scales on {scales.device}")
        self.data, self.scales, self.dim, self.dtype = _aligned(data), _aligned(scales), dim, dtype

    @property
    def shape(self):
        return torch.Size((*self.data.shape[:-1], self.dim))

    @property
    def device(self):
        return self.data.device

    def get_device(self):
        return self.data.get_device()

    @property
    def rows(self) -> int:
        return self.data.numel() // self.data.shape[-1]

    @staticmethod
    def _empty(shape, like, dtype):
        m = object.__new__(Mx8)
        m.dim, m.dtype = shape[-1], dtype
        m.data = torch.empty((*shape[:-1], 32 * -(-m.dim // 32)), dtype=torch.float8_e4m3fn, device=like.device)
        m.scales = torch.empty((*shape[:-1], 4 * -(-m.dim // 128)), dtype=torch.uint8, device=like.device)
        return m


def _aligned(t):
    """t contiguous from a 16-byte boundary on."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _mx8_rows(lib, call, matrix, dim, m, like):
    a = _abi.Mx8Args(_stream(like), matrix.shape[0], dim, _dtype(matrix), matrix.data_ptr(), matrix.stride(0),
                     m.data.data_ptr(), m.scales.data_ptr())
    _abi.check(call(ctypes.byref(a)))


def mx8_pack(x) -> Mx8:
    """x in 8 bits: each 32 adjacent columns share a power of two, and a number is
    kept to within 1/16 of itself, or 2^-17 of its block's largest (and 2^-136) where
    that is more.  Infinities and NaN become NaN; float16 beyond 61440 (the others beyond
    3.19e38) count as that."""
    lib, _ = _library(x), _dtype(x)
    x2 = _feature_rows("x", x)
    m = Mx8._empty(x.shape, x, x.dtype)
    _mx8_rows(lib, lib.msplat_hip_mx8_pack, x2, x2.shape[1], m, x)
    return m


def mx8_unpack(m: Mx8, dtype=None):
    """The numbers that m holds, in its own type or `dtype` (exact but where the
    type is float16 and they pass its range)."""
    lib, dtype = _library(m), dtype or m.dtype
    if dtype not in _DTYPES:
        raise ValueError(f"{dtype} is none of float32, float16, bfloat16")
    y = torch.empty(m.shape, dtype=dtype, device=m.device)
    _mx8_rows(lib, lib.msplat_hip_mx8_unpack, y.view(-1, m.dim) if y.numel() else y.new_empty(0, m.dim), m.dim, m, y)
    return y


def rms_norm_forward(x, weight=None, residual=None, eps: float = 1e-5, mx8: bool = False):
    """(y, total, rstd): total = x + residual of x's type (x itself without a
    residual), y = total rstd weight over the last axis, rstd = 1 / sqrt(mean(total^2)
    + eps), one float32 a row.  mx8: y is an Mx8, rounded to 8 bits once.  A sum of squares
    beyond float32 counts as infinite (rstd 0)."""
    lib, dtype = _library(x), _dtype(x)
    x2 = _feature_rows("x", x)
    rows, dim = x2.shape
    r2 = None if residual is None else _same_rows("residual", residual, x2)
    w = None if weight is None else _matrix("weight", weight, (dim,), x)
    y = Mx8._empty(x.shape, x, x.dtype) if mx8 else x.new_empty(x.shape)
    total = x if residual is None else x.new_empty(x.shape)
    rstd = x.new_empty(x.shape[:-1], dtype=torch.float32)
    a = _abi.RmsNormArgs(_stream(x), rows, dim, dtype, x2.data_ptr(), x2.stride(0), _ptr(r2),
                         0 if r2 is None else r2.stride(0), _ptr(w), eps, (y.data if mx8 else y).data_ptr(), dim,
                         y.scales.data_ptr() if mx8 else None, None if residual is None else total.data_ptr(), dim,
                         rstd.data_ptr())
    _abi.check(lib.msplat_hip_rms_norm(ctypes.byref(a)))
    return y, total, rstd


def rms_norm_backward(dy, total, weight, rstd, dtotal=None, wanted=(True, True)):
    """(dx, dweight) from the gradients of y and (where not None) of total, and the
    forward's total, a tensor or an Mx8 of it, and rstd.  dx is the gradient of x
    and of residual alike; dweight has dy's type, also where weight is None.
    Those not wanted are None and not computed."""
    lib, dtype = _library(dy), _dtype(dy)
    dy2 = _feature_rows("dy", dy)
    rows, dim = dy2.shape
    if isinstance(total, Mx8):
        ts = _mx8_operand("total", total, rows, dim, dy)
    else:
        t2 = _same_rows("total", total, dy2)
        ts = (t2.data_ptr(), t2.stride(0), None)
    g2 = None if dtotal is None else _same_rows("dtotal", dtotal, dy2)
    w = None if weight is None else _matrix("weight", weight, (dim,), dy)
    if rstd.dtype is not torch.float32 or rstd.numel() != rows or rstd.device != dy.device:
        raise ValueError(f"rstd must hold one float32 a row on {dy.device}")
    rstd = rstd.contiguous()
    dx = dy.new_empty(dy.shape) if wanted[0] else None
    dweight = dy.new_empty(dim) if wanted[1] else None
    ws = _workspace(lib.msplat_hip_rms_norm_backward_workspace(rows, dim, dtype), dy) if wanted[1] else None
    a = _abi.RmsNormGradArgs(_stream(dy), rows, dim, dtype, dy2.data_ptr(), dy2.stride(0), _ptr(g2),
                             0 if g2 is None else g2.stride(0), *ts, _ptr(w),
                             rstd.data_ptr(), _ptr(dx), dim, _ptr(dweight), _ptr(ws), 0 if ws is None else ws.nbytes)
    _abi.check(lib.msplat_hip_rms_norm_backward(ctypes.byref(a)))
    return dx, dweight


_LINEAR_ACTIVATIONS = {"silu": 0, "gelu": 1, None: 2}
_MX8 = 3   # MSPLAT_MX8


def _linear_activation(activation) -> int:
    if activation not in _LINEAR_ACTIVATIONS:
        raise ValueError(f"activation {activation!r} is none of None, 'silu', 'gelu'")
    return _LINEAR_ACTIVATIONS[activation]


def linear_forward(x, weight, bias=None, residual=None, activation=None, out_dtype=None, keep: bool = False):
    """residual + a(x weight^T + bias) with a = None (the identity), "silu" or "gelu"
    (tanh form); weight [outer, inner], bias [outer].  x and weight are of one type, as
    is bias, or both Mx8 with a float32 bias.  The result and residual have `out_dtype`,
    x's own where None.  keep: (result, x weight^T + bias in x's type, in float16 to
    65504 at most), the latter for the backward.  A row of x that holds an infinity may come out as NaN
    throughout; other rows are untouched."""
    act = _linear_activation(activation)
    kept = isinstance(x, Mx8)
    if kept is not isinstance(weight, Mx8):
        raise ValueError("x and weight are both Mx8 or neither is")
    lib, out_dtype = _library(x), out_dtype or x.dtype
    if out_dtype not in _DTYPES:
        raise ValueError(f"{out_dtype} is none of float32, float16, bfloat16")
    if kept:
        if keep:
            raise ValueError("a product of Mx8 has no backward to keep anything for")
        rows, inner, outer, like = x.rows, x.dim, weight.rows, x.data
        if weight.data.dim() != 2 or weight.dim != inner or weight.device != x.device:
            raise ValueError(f"weight has shape {tuple(weight.shape)} on {weight.device}, not [outer, {inner}] on "
                             f"{x.device}")
        dtype, b = _MX8, None if bias is None else _vector("bias", bias, outer, torch.float32, x.device)
        ops = (x.data.data_ptr(), 0, x.scales.data_ptr(), weight.data.data_ptr(), 0, weight.scales.data_ptr())
    else:
        x2, like, dtype = _feature_rows("x", x), x, _dtype(x)
        rows, inner = x2.shape
        if weight.dim() != 2:
            raise ValueError(f"weight has shape {tuple(weight.shape)}, not (outer, {inner})")
        outer = weight.shape[0]
        w = _matrix("weight", weight, (outer, inner), x)
        b = None if bias is None else _matrix("bias", bias, (outer,), x)
        ops = (x2.data_ptr(), x2.stride(0), None, w.data_ptr(), w.stride(0), None)
    shape = (*x.shape[:-1], outer)
    y = like.new_empty(shape, dtype=out_dtype)
    r2 = None if residual is None else _rows_of("residual", residual, rows, outer, y)
    z = like.new_empty(shape) if keep else None
    nbytes = lib.msplat_hip_linear_workspace(rows, inner, outer, dtype)
    ws = _workspace(nbytes, y) if nbytes else None
    a = _abi.LinearArgs(_stream(like), rows, inner, outer, dtype, _DTYPES[out_dtype], act, *ops, _ptr(b), _ptr(r2),
                        0 if r2 is None else r2.stride(0), y.data_ptr(), outer, _ptr(z), outer, _ptr(ws),
                        0 if ws is None else ws.nbytes)
    _abi.check(lib.msplat_hip_linear(ctypes.byref(a)))
    return (y, z) if keep else y


def linear_backward(dy, x, weight, z=None, activation=None, wanted=(True, True, True)):
    """(dx, dweight, dbias) from the gradient of the result, x, weight and, where there
    is an activation, what the forward kept; x and z may be Mx8 of them.  The
    gradients have weight's type.  Those not wanted are None and not computed; without
    dweight x may be None.  In 16-bit types dy a'(z), also of a dy in float32, is rounded
    to the type for dx and dweight (float16: fewer bits below 6e-5, 0 below 3e-8, infinite
    beyond 65504).  A row of dy that holds an infinity may make its row of dx NaN
    throughout; other rows are untouched."""
    act = _linear_activation(activation)
    if x is None and wanted[1]:
        raise ValueError("the weight's gradient takes x")
    _tensor("weight", weight)
    lib, dtype = _library(weight), _dtype(weight)
    if weight.dim() != 2 or min(weight.shape) < 1:
        raise ValueError(f"weight has shape {tuple(weight.shape)}, not (outer, inner)")
    outer, inner = weight.shape
    w = _matrix("weight", weight, (outer, inner), weight)
    dy2 = _rows("dy", dy, outer, dy)
    rows = dy2.shape[0]
    if x is None:
        xs = (None, 0, None)
    elif isinstance(x, Mx8):
        xs = _mx8_operand("x", x, rows, inner, weight)
    else:
        x2 = _rows_of("x", x, rows, inner, weight)
        xs = (x2.data_ptr(), x2.stride(0), None)
    if dy.device != weight.device:
        raise ValueError(f"dy is on {dy.device}, not {weight.device}")
    if activation is None:
        zs = (None, 0, None)
    elif isinstance(z, Mx8):
        zs = _mx8_operand("z", z, rows, outer, weight)
    elif z is None:
        raise ValueError("the backward of an activation takes z")
    else:
        z2 = _rows_of("z", z, rows, outer, weight)
        zs = (z2.data_ptr(), z2.stride(0), None)
    dx = weight.new_empty((*dy.shape[:-1], inner) if x is None else x.shape) if wanted[0] else None
    dweight = weight.new_empty(outer, inner) if wanted[1] else None
    dbias = weight.new_empty(outer) if wanted[2] else None
    ws = _workspace(lib.msplat_hip_linear_backward_workspace(rows, inner, outer, dtype, _dtype(dy), act), weight)
    a = _abi.LinearGradArgs(_stream(weight), rows, inner, outer, dtype, _dtype(dy), act, dy2.data_ptr(), dy2.stride(0),
                            *xs, w.data_ptr(), w.stride(0), *zs, _ptr(dx), inner, _ptr(dweight), _ptr(dbias),
                            ws.data_ptr(), ws.nbytes)
    _abi.check(lib.msplat_hip_linear_backward(ctypes.byref(a)))
    return dx, dweight, dbias


def _vector(name, t, n, dtype, dev):
    if t.dtype is not dtype or t.device != dev or tuple(t.shape) != (n,):
        raise ValueError(f"{name} is {t.dtype} of shape {tuple(t.shape)} on {t.device}, not {dtype} of ({n},) on {dev}")
    return t.contiguous()


def _rows_of(name, t, rows, dim, like):
    t2 = _rows(name, t, dim, like)
    if t2.shape[0] != rows:
        raise ValueError(f"{name} has {t2.shape[0]} rows, not {rows}")
    return t2


def _mx8_operand(name, m, rows, dim, like):
    if m.dim != dim or m.rows != rows:
        raise ValueError(f"{name} has shape {tuple(m.shape)}, not {rows} rows of {dim}")
    if m.device != like.device or m.dtype is not like.dtype:
        raise ValueError(f"{name} stands for {m.dtype} on {m.device}, not {like.dtype} on {like.device}")
    return m.data.data_ptr(), 0, m.scales.data_ptr()


_CHECKPOINTS = (None, "mx8")


def _check_checkpoint(checkpoint):
    if checkpoint not in _CHECKPOINTS:
        raise ValueError(f"checkpoint {checkpoint!r} is none of {_CHECKPOINTS}")


def _smaller_packed(t) -> bool:
    """Whether a matrix takes less room in 8 bits: a row of those has whole blocks
    of 32 columns (5 columns of float32: 36 bytes instead of 20)."""
    dim = t.shape[-1]
    return 32 * -(-dim // 32) + 4 * -(-dim // 128) < dim * t.element_size()


def _keep(ctx, checkpoint, kept, *others):
    """Saves tensors for the backward, those in `kept` (each may be None) as
    Mx8 where the checkpoint says so and that is smaller."""
    if checkpoint is None:
        ctx.kept = None
        return ctx.save_for_backward(*kept, *others)
    packed = [mx8_pack(t) if t is not None and _smaller_packed(t) else t for t in kept]
    ctx.kept = [(m.dim, m.dtype) if isinstance(m, Mx8) else None for m in packed]
    flat = [t for m in packed for t in ((m.data, m.scales) if isinstance(m, Mx8) else (m, None))]
    ctx.save_for_backward(*flat, *others)


def _kept(ctx):
    """What _keep took: those that it kept, and the others."""
    saved = ctx.saved_tensors
    if ctx.kept is None:
        return saved
    n = len(ctx.kept)
    pairs = [Mx8(*saved[2 * i:2 * i + 2], *k) if k else saved[2 * i] for i, k in enumerate(ctx.kept)]
    return [*pairs, *saved[2 * n:]]


def _shaped(g, shape):
    """g as the gradient of an input of that shape.  Autograd makes a gradient that
    nobody else holds a leaf's own, and looks at the tensor, not at its memory: g itself
    where the shape is its own, and never a view, whose memory is another gradient's or the
    caller's."""
    return g if g.shape == shape else g.clone(memory_format=torch.contiguous_format).view(shape)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        return (*layer_norm_backward(dy, x, weight, mean, rstd, ctx.needs_input_grad[:3]), None)


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation, checkpoint, grad):
        y = gated_ffn_forward(x, w_gate, w_up, w_down, activation)
        if grad and any(ctx.needs_input_grad[:4]):
            _keep(ctx, checkpoint, (x,), w_gate, w_up, w_down)
            ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        x, *weights = _kept(ctx)
        x = mx8_unpack(x) if isinstance(x, Mx8) else x
        dx, *grads = gated_ffn_backward(dy, x, *weights, ctx.activation, (need[0], any(need[1:4])))
        return (dx, *(g if n else None for g, n in zip(grads, need[1:4])), None, None, None)


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        ctx.args = (p, seed, offset)
        ctx.residual_shape = None if residual is None else residual.shape
        if torch.is_tensor(offset):   # saved, so that a change before the backward is an error
            ctx.args = (p, seed)
            ctx.save_for_backward(offset)
        return dropout_add_forward(x, residual, p, seed, offset)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        dx = dropout_add_backward(dy, *ctx.args, *ctx.saved_tensors) if need[0] else None
        return dx, _shaped(dy, ctx.residual_shape) if need[1] else None, None, None, None


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, checkpoint, grad):
        ctx.set_materialize_grads(False)
        y, total, rstd = rms_norm_forward(x, weight, residual, eps)
        if grad and any(ctx.needs_input_grad[:3]):
            ctx.residual_shape = None if residual is None else residual.shape
            _keep(ctx, checkpoint, (total,), weight, rstd)
        return y if residual is None else (y, total)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dtotal=None):
        if dy is None and dtotal is None:   # no gradient reaches either result
            return (None,) * 6
        total, weight, rstd = _kept(ctx)
        need = ctx.needs_input_grad
        along = need[0] or need[2]
        if dy is None:   # y was not used
            dweight = None if weight is None or not need[1] else torch.zeros_like(weight)
            dx = dtotal
        else:
            dx, dweight = rms_norm_backward(dy, total, weight, rstd, dtotal, (along, need[1]))
        return dx if need[0] else None, dweight, _shaped(dx, ctx.residual_shape) if need[2] else None, None, None, None


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, out_dtype, checkpoint, grad):
        need = ctx.needs_input_grad
        keep = grad and activation is not None and any(need[:3])
        y = linear_forward(x, weight, bias, residual, activation, out_dtype, keep)
        y, z = y if keep else (y, None)
        ctx.activation = activation
        ctx.residual_shape = None if residual is None else residual.shape
        if grad and any(need[:3]):
            _keep(ctx, checkpoint, (x if need[1] else None, z), weight)   # x is for the weight's gradient alone
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        grads = None, None, None
        if any(need[:3]):
            x, z, weight = _kept(ctx)
            grads = linear_backward(dy, x, weight, z, ctx.activation, need[:3])
        return (*grads, _shaped(dy, ctx.residual_shape) if need[3] else None, None, None, None, None)


def _no_derivatives(grad) -> bool:
    """Whether a call may go past autograd, which takes 3 us: without gradients, and outside
    forward mode, whose tangents autograd refuses whatever the grad mode is."""
    return not grad and forward_ad._current_level < 0


def linear(x, weight, bias=None, residual=None, activation=None, out_dtype=None, checkpoint=None):
    """linear_forward, differentiable in x, weight, bias and residual.  checkpoint
    "mx8" keeps x and x weight^T + bias for the backward in 8 bits, where that is less.
    A float16 weight's backward rounds the result's gradient to float16, whatever
    out_dtype is: scale the loss so that it stays above 6e-5, or use bfloat16."""
    _check_checkpoint(checkpoint)
    if isinstance(x, Mx8) or isinstance(weight, Mx8):
        raise ValueError("a product of Mx8 has no gradients: call linear_forward")
    grad = torch.is_grad_enabled()   # off in an autograd function's forward
    if _no_derivatives(grad):
        return linear_forward(x, weight, bias, residual, activation, out_dtype)
    return _Linear.apply(x, weight, bias, residual, activation, out_dtype, checkpoint, grad)


def rms_norm(x, weight=None, residual=None, eps: float = 1e-5, checkpoint=None):
    """rms_norm_forward's y, and with a residual (y, total), differentiable in x,
    weight and residual.  checkpoint "mx8" keeps total for the backward in 8 bits, where
    that is less."""
    _check_checkpoint(checkpoint)
    grad = torch.is_grad_enabled()
    if _no_derivatives(grad):
        y, total, _ = rms_norm_forward(x, weight, residual, eps)
        return y if residual is None else (y, total)
    return _RmsNorm.apply(x, weight, residual, eps, checkpoint, grad)


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """layer_norm_forward's y, differentiable in x, weight and bias."""
    return _LayerNorm.apply(x, weight, bias, eps)


def gated_ffn(x, w_gate, w_up, w_down, activation: str = "silu", checkpoint=None):
    """gated_ffn_forward, differentiable in x and the three weights.  checkpoint
    "mx8" keeps x for the backward in 8 bits, where that is less."""
    _check_checkpoint(checkpoint)
    return _GatedFfn.apply(x, w_gate, w_up, w_down, activation, checkpoint, torch.is_grad_enabled())


def dropout_add(x, residual, p: float, seed: int, offset):
    """dropout_add_forward, differentiable in x and residual.  An offset tensor
    must keep its value until the backward has run."""
    return _DropoutAdd.apply(x, residual, p, seed, offset)
