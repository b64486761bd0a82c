"""Operators of a learned head, trained next to a scene.

Layer norm, a gated feed-forward block and dropout added to a residual, over
the features of gaussians or pixels: CUDA tensors [..., dim] of float32,
float16 or bfloat16 (one type a call), with any stride between rows, on the GPU
of the library's context (the first call's, if none has made one yet).  Each
runs hand-written kernels of libmsplat_hip.so on PyTorch's current stream, sums
in fp32, and has

  layer_norm, gated_ffn, dropout_add          differentiable by autograd
  *_forward, *_backward                       the two passes by themselves

None of them waits for the GPU or keeps anything between calls, so they may
be captured into a graph.  A replay repeats a call's arguments: where each is to
drop other elements, dropout takes its offset as a tensor.
"""
from __future__ import annotations

import ctypes
from operator import index   # numpy's integers overflow in & where Python's do not
from typing import Tuple

import torch
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


def _rows(name, t, dim, like):
    """t as a [rows, dim] matrix with adjacent columns."""
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
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        ctx.save_for_backward(x, w_gate, w_up, w_down)
        ctx.activation = activation
        return gated_ffn_forward(x, w_gate, w_up, w_down, activation)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        dx, *grads = gated_ffn_backward(dy, *ctx.saved_tensors, ctx.activation, (need[0], any(need[1:4])))
        return (dx, *(g if n else None for g, n in zip(grads, need[1:4])), None)


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        ctx.args = (p, seed, offset)
        if torch.is_tensor(offset):   # saved, so that a change before the backward is an error
            ctx.args = (p, seed)
            ctx.save_for_backward(offset)
        return dropout_add_forward(x, residual, p, seed, offset)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        dx = dropout_add_backward(dy, *ctx.args, *ctx.saved_tensors) if need[0] else None
        return dx, dy if need[1] else None, None, None, None


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """layer_norm_forward's y, differentiable in x, weight and bias."""
    return _LayerNorm.apply(x, weight, bias, eps)


def gated_ffn(x, w_gate, w_up, w_down, activation: str = "silu"):
    """gated_ffn_forward, differentiable in x and the three weights."""
    return _GatedFfn.apply(x, w_gate, w_up, w_down, activation)


def dropout_add(x, residual, p: float, seed: int, offset):
    """dropout_add_forward, differentiable in x and residual.  An offset tensor
    must keep its value until the backward has run."""
    return _DropoutAdd.apply(x, residual, p, seed, offset)
