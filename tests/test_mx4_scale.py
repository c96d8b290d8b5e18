"""Attention's scale is a number: what is none is refused before anything is done."""

import ctypes
import math

import pytest
import torch

from sparseflow_amd import _lib
from sparseflow_amd.Kernels.cached_attention import cached_attention_forward, cached_attention_step, mx4_cache
from sparseflow_amd.Ops import CachedAttention


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 2.0 ** 127, torch.tensor(math.nan)], ids=str)
def test_scales_that_are_refused(scale):
    cache = mx4_cache(2, 1, 8, 32)
    tables, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.randn(1, 1, 2, 32)
    with pytest.raises(ValueError):
        cached_attention_forward(q, cache, tables, lengths, scale=scale)
    with pytest.raises(ValueError):
        cached_attention_step(q[:, 0], cache, tables, lengths, scale=scale)
    with pytest.raises(ValueError):
        CachedAttention(scale=scale)


@pytest.mark.parametrize("scale", [0.0, -2.0, 2.0 ** 126, torch.tensor(0.5)], ids=str)
def test_scales_that_are_taken(scale):
    cache = mx4_cache(2, 1, 8, 32)
    tables, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    y = cached_attention_forward(torch.randn(1, 1, 2, 32), cache, tables, lengths, scale=scale)
    assert not y.any()  # (values of 0)


def test_scales_of_the_c_abi():
    L = _lib.lib()
    one, at, zero = ctypes.c_void_p(16), ctypes.addressof, (0, 0, 0)
    t = _lib.Mx4CacheTensors(16, 16, 16, 16, 16, 16)
    for scale in (math.nan, math.inf, -math.inf, 2.0 ** 127):
        c = _lib.Mx4CacheDesc(1, 1, 1, 1, 1, 1, zero, zero, zero, zero, 4, 2, 20, 8, 0, scale)
        assert L.sf_mx4_attention(at(c), at(t), one, None, None, one, None, 0, None) == _lib.SF_ERR_INVALID
