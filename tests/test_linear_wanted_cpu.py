"""Gradients of the linear layer that do not take its input, without a GPU: what the
C entry point and msplat_amd.nn ask for."""
from __future__ import annotations

import ctypes

import pytest
import torch

from msplat_amd import nn
from test_more_cpu import _linear_grad
from test_nn_cpu import lib  # noqa: F401


def test_x_is_needed_for_the_weights_gradient_alone(lib):  # noqa: F811
    from msplat_amd import device
    if device._initialised:
        pytest.skip("a context already exists in this process")
    for kw in (dict(x=None), dict(x=None, x_stride=0), dict(x=None, dbias=None), dict(x=None, dx=None)):
        _, a = _linear_grad(**kw)
        assert lib.msplat_hip_linear_backward(ctypes.byref(a)) == -1 and b"x is null" in lib.msplat_hip_last_error()
        a.dweight = None
        assert lib.msplat_hip_linear_backward(ctypes.byref(a)) == -3   # no context


def test_python_says_so():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="takes x"):
        nn.linear_backward(x, None, x)
