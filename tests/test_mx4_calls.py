"""Calls of the 4-bit entry points that repeat with other numbers: nothing is kept by a tensor's identity."""

import torch

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
