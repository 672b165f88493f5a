"""The device of a handle comes from the library: it needs no torch, whatever torch there is, and tensors on other devices are
refused. On a stand-in for the library, so without a GPU."""
import ctypes

import pytest

import hiptensor_b200 as ht
from hiptensor_b200 import _lib


class Library:
    """Hands out a handle on device 3 and takes every call."""

    def __init__(self):
        self.calls = []

    def htGetErrorString(self, status):
        return b"status %d" % status

    def htCreate(self, out):
        ctypes.cast(out, ctypes.POINTER(ctypes.c_void_p))[0] = 4096
        return 0

    def htGetDevice(self, handle, out):
        assert handle.value == 4096
        ctypes.cast(out, ctypes.POINTER(ctypes.c_int32))[0] = 3
        return 0

    def htDestroy(self, handle):
        return 0

    def htCrossEntropy(self, *args):
        self.calls.append(args)
        return 0


class Tensor:
    def __init__(self, device):
        self.device = device

    def get_device(self):
        return self.device

    def data_ptr(self):
        return 256 * (self.device + 2)


@pytest.fixture
def library(monkeypatch):
    L = Library()
    monkeypatch.setattr(_lib, "lib", lambda: L)
    return L


class Plan:
    _p = ctypes.c_void_p(0)


def call(h, x):
    h.cross_entropy(Plan(), 1.0, x, 512, 512, 512, 512, 512, 512)


def test_a_torch_that_has_no_device_does_not_matter(library, monkeypatch):
    torch = pytest.importorskip("torch")

    def none():
        raise AssertionError("Torch not compiled with CUDA enabled")

    monkeypatch.setattr(torch.cuda, "current_device", none)
    h = ht.Handle()
    call(h, Tensor(3))
    assert len(library.calls) == 1


def test_tensors_on_another_device_are_refused_without_torch_too(library, monkeypatch):
    import sys

    monkeypatch.delitem(sys.modules, "torch", raising=False)  # not imported yet when the handle was made
    h = ht.Handle()
    for device in (-1, 0, 2):
        with pytest.raises(ht.HiptensorError) as e:
            call(h, Tensor(device))
        assert e.value.status == ht.STATUS_ARCH_MISMATCH
    call(h, Tensor(3))
    assert len(library.calls) == 1


def test_no_handle_no_device():
    from hiptensor_b200 import build

    build.build()
    L, out = _lib.lib(), ctypes.c_int32(-1)
    assert L.htGetDevice(None, ctypes.byref(out)) == ht.STATUS_NOT_INITIALIZED
    blank = ctypes.create_string_buffer(1 << 12)
    assert L.htGetDevice(ctypes.addressof(blank), ctypes.byref(out)) == ht.STATUS_NOT_INITIALIZED and out.value == -1
