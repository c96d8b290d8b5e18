"""Attention over the 4-bit cache on the GPU: numbers that are none, where the tokens are cut into parts."""

import math

import pytest
import torch

from sparseflow_amd.Kernels.cached_attention import MX4Cache, cached_attention_forward
from tests.gpu_helpers import DEV, announce
from tests.mx4_checks import attention_case

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("n", [1, 60])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf], ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_queries_that_are_none(dtype, value, n):
    """A NaN in a query makes its row NaN in every part, and so does an infinity: of 4000 tokens' codes some are 0."""
    announce(f"attention none {dtype} {value} {n}")
    call, _, _ = attention_case(DEV, [n, n], [4000, 700], 4, 2, 64, 16, dtype, False)
    base = cached_attention_forward(**call)
    q = call["q"].clone()
    q[:, n // 2, 1, 5] = value
    y = cached_attention_forward(**{**call, "q": q})
    hit = torch.zeros(2, n, 4, dtype=torch.bool, device=DEV)
    hit[:, n // 2, 1] = True
    assert torch.isnan(y[hit]).all()
    assert torch.equal(y[~hit], base[~hit])


@pytest.mark.parametrize("n", [1, 60])
@pytest.mark.parametrize("first,last", [(0, 4000), (512, 1024), (512, 768), (512, 800), (1000, 1001)])
@pytest.mark.parametrize("dtype", TYPES)
def test_runs_of_keys_that_are_none(dtype, first, last, n):
    """Every query sees some of them, beside others; runs that are whole parts, and that are not."""
    announce(f"attention keys none {dtype} {first} {last} {n}")
    call, _, _ = attention_case(DEV, [n], [4000], 4, 2, 64, 16, dtype, False)
    base = cached_attention_forward(**call)
    cache = MX4Cache(*(t.clone() for t in call["cache"]))
    t = torch.arange(first, last, device=DEV)
    cache.k_scales[call["tables"][0, t // 16].long(), 1, t % 16, 0] = 255
    y = cached_attention_forward(**{**call, "cache": cache})
    assert torch.isnan(y[:, :, 2:]).all() and torch.equal(y[:, :, :2], base[:, :, :2])
