"""How msplat_amd.nn calls the library, without a GPU: stand-ins for tensors and
for the library.  And the widths that the library takes."""
from __future__ import annotations

import contextlib
import ctypes
import os

import pytest
import torch

import msplat_amd
from msplat_amd import _abi, device, nn


class _On:
    """A tensor on GPU `index`, as far as the operators look before they call."""

    is_cuda = True
    dtype = torch.float32

    def __init__(self, index):
        self.device = torch.device("cuda", index)

    def get_device(self):
        return self.device.index


@pytest.fixture
def context(monkeypatch):
    """A context on GPU 0."""
    library = object()
    monkeypatch.setattr(device, "_initialised", True)
    monkeypatch.setattr(device, "_lib", library, raising=False)
    monkeypatch.setattr(device, "_device", 0, raising=False)
    monkeypatch.setattr(device._abi, "load", lambda: library)
    return library


def test_another_gpus_tensors_are_refused(context):
    assert nn._library(_On(0)) is context
    far = _On(1)
    for call in (lambda: nn._library(far), lambda: nn.layer_norm_forward(far),
                 lambda: nn.gated_ffn_forward(far, *[far] * 3), lambda: nn.dropout_add_forward(far, None, 0.5, 1, 2)):
        with pytest.raises(ValueError, match="cuda:1"):
            call()


def test_the_first_call_leaves_the_current_device(monkeypatch):
    """The context is made on the tensors' GPU, in a guard of PyTorch's, and again
    after a cleanup."""
    seen = []

    @contextlib.contextmanager
    def guard(index):
        seen.append(("enter", index))
        yield
        seen.append("leave")

    class Library:
        def msplat_hip_init(self, index):
            seen.append(("init", index))
            return 0

        def msplat_hip_shutdown(self):
            seen.append("cleanup")
            return 0

    library = Library()
    monkeypatch.setattr(device, "_initialised", False)
    monkeypatch.setattr(device, "_lib", None, raising=False)
    monkeypatch.setattr(device, "_device", None, raising=False)
    monkeypatch.setattr(device._abi, "load", lambda: library)
    monkeypatch.setattr(torch.cuda, "device", guard)
    assert nn._library(_On(3)) is library
    assert seen == [("enter", 3), ("init", 3), "leave"]
    msplat_amd.cleanup()
    assert nn._library(_On(2)) is library
    assert seen[3:] == ["cleanup", ("enter", 2), ("init", 2), "leave"]


def test_the_widest_dropout():
    """Refused from 2^31 - 255 columns on; the widest goes on to the missing context."""
    if not os.path.exists(_abi.LIB_PATH):
        pytest.skip("libmsplat_hip.so not built")
    if device._initialised:
        pytest.skip("a context already exists in this process")
    lib = _abi.load()
    host = (ctypes.c_double * 2)()
    at = ctypes.addressof(host)
    for dim, code in ((2 ** 31 - 256, -3), (2 ** 31 - 255, -1)):
        a = _abi.DropoutArgs(None, 1, dim, 2, 0.5, 1, 2, at, dim, None, 0, at, dim)
        assert lib.msplat_hip_dropout_add(ctypes.byref(a)) == code


def test_offsets_in_memory_are_checked():
    if not os.path.exists(_abi.LIB_PATH):
        pytest.skip("libmsplat_hip.so not built")
    lib = _abi.load()
    host = (ctypes.c_double * 8)()
    at = ctypes.addressof(host)
    a = _abi.DropoutArgs(None, 1, 4, 0, 0.5, 1, 2, at, 4, None, 0, at, 4)
    for offset, word in ((None, b"offset is null"), (at + 4, b"aligned")):
        assert lib.msplat_hip_dropout_add_at(ctypes.byref(a), offset) == -1
        assert word in lib.msplat_hip_last_error()
    assert lib.msplat_hip_dropout_add_at(None, at) == -1
    a.dim = 0
    assert lib.msplat_hip_dropout_add_at(ctypes.byref(a), at) == -1 and b"dim" in lib.msplat_hip_last_error()
