"""Calls of the 4-bit entry points that repeat with other numbers: nothing is kept by a tensor's identity."""

import ctypes
import gc

import torch

from sparseflow_amd import _lib
from sparseflow_amd.Kernels.mx4 import mx4_dequantize, mx4_quantize


def test_a_size_that_comes_as_a_tensor_is_read_at_every_call():
    x = torch.randn(3, 40)
    q = mx4_quantize(x)
    size = torch.tensor(40)
    whole = mx4_dequantize(*q, size=size)
    assert whole.shape == (3, 40)
    size.fill_(33)
    assert torch.equal(mx4_dequantize(*q, size=size), whole[:, :33])
    size.fill_(64)
    assert torch.equal(mx4_dequantize(*q, size=size)[:, :40], whole)


def test_strides_live_as_long_as_the_call(monkeypatch):
    """What a call's address points to is held by the call, not only by a cache that other threads may empty."""
    held = []

    def launch(name, device, *args):
        _lib._pair.cache_clear()
        at = args[4]
        held.append([list(o) for o in gc.get_objects() if type(o) is ctypes.c_int64 * 2 and ctypes.addressof(o) == at])

    monkeypatch.setattr(_lib, "_launch", launch)
    x = torch.randn(3, 40)
    _lib.mx4_quantize(x, 1, 3, (0, 40), torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(3, 2, dtype=torch.uint8))
    assert held == [[[0, 40]]]
