"""Attention over the 4-bit cache on the GPU: values of any magnitude that float32 has."""

import pytest
import torch

from oracle import mx4 as ora
from sparseflow_amd.Kernels.cached_attention import cached_attention_forward, mx4_cache, mx4_cache_append
from tests.gpu_helpers import DEV, announce
from tests.mx4_checks import PARTS, STEP, half_step, within

pytestmark = pytest.mark.gpu


def _check(dtype, n, old, magnitudes, what):
    """magnitudes [tokens]: the powers of two that a token's values have.  The bound: a weight's relative error (two of a
    score's, the exponential's, its parts'), a step of the magnitudes' sum to each term of both sums, half a step of the
    result, and for each of a token's three terms float32's smallest number, 2^-149, over the sum of the weights, 1/2 at
    least.  Where values from 2^95 on are about, weights have 2^-30 as a factor, and so has that sum."""
    g = torch.Generator().manual_seed(n + old)
    dim, page, total = 64, 16, n + old
    width = -(-total // page)
    tables = torch.randperm(width, generator=g).int()[None].to(DEV)
    lengths = torch.tensor([total], dtype=torch.int32, device=DEV)
    k = torch.randn(1, total, 1, dim, generator=g)
    v = torch.randn(1, total, 1, dim, generator=g) * torch.exp2(magnitudes.float())[None, :, None, None]
    q = torch.randn(1, n, 2, dim, generator=g).to(dtype)
    cache = mx4_cache(width, 1, page, dim, device=DEV)
    mx4_cache_append(cache, k.to(dtype).to(DEV), v.to(dtype).to(DEV), tables, lengths)
    rows = tables[0].long()
    held = [ora.values(c[rows, 0].flatten(0, 1)[:total], s[rows, 0].flatten(0, 1)[:total], dim)
            for c, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales))]
    assert torch.isfinite(held[1]).all()
    y = cached_attention_forward(q.to(DEV), cache, tables, lengths)
    see = torch.arange(total)[None] <= (torch.arange(n) + old)[:, None]
    parts = PARTS[dtype]
    lost = 2.0 ** (-118 if bool((held[1].abs() >= 2.0 ** 94).any()) else -148)
    for h in range(2):
        ref, mag, big = ora.attend(q[0, :, h], *held, see, dim ** -0.5)
        score = (parts * dim + 8) * STEP * big * 1.5
        weight = 2 * score + 8 * STEP + (0.0 if parts == 3 else 2.0 ** -16)
        bound = mag * (weight[:, None] + (3 * total + 8) * 2 * STEP) + half_step(dtype) * ref.abs() + 3 * total * lost
        within(y[0, :, h], ref, bound, what)


@pytest.mark.parametrize("n,old", [(1, 45), (60, 45), (1, 3000), (60, 3000)])
@pytest.mark.parametrize("power", [-118, -105, -97, -60, 60, 93, 95, 120])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_of_one_magnitude(dtype, power, n, old):
    announce(f"value range {dtype} {power} {n} {old}")
    _check(dtype, n, old, torch.full((n + old,), power), f"2^{power}")


@pytest.mark.parametrize("n,old", [(1, 45), (60, 45), (1, 3000), (60, 3000)])
@pytest.mark.parametrize("power", [93, 97, 120])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_that_grow(dtype, power, n, old):
    """Ordinary values, and one token, in the first, a middle and the last part of them, of large ones."""
    announce(f"value range grows {dtype} {power} {n} {old}")
    for at in (0, (n + old) // 2, n + old - 1):
        magnitudes = torch.zeros(n + old)
        magnitudes[at] = power
        _check(dtype, n, old, magnitudes, f"2^{power} at {at}")
