"""Attention over the 4-bit cache on the GPU: softmax weights are held to more than a result's bits."""

import math

import pytest
import torch

from oracle import mx4 as ora
from sparseflow_amd.Kernels.cached_attention import cached_attention_forward, mx4_cache, mx4_cache_append
from tests.gpu_helpers import DEV, announce
from tests.mx4_checks import STEP, half_step, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_weights_of_sums_that_cancel(dtype, n):
    """Sixteen tokens of weight 1 against sixteen of weight w, whose values nearly cancel: what a weight loses is all there is
    to see.  Two parts of 8 bits are off by 2^-16 of a weight (the first is cut off, less than 2^-7 is left, and of that half
    a step of 8 bits, 2^-9, is lost); a score by few steps (one product and the scale), the exponential by 2^-22, 32 tokens'
    sums by a step each of both parts, twice (the sum of the weights too)."""
    announce(f"attention weights {dtype} {n}")
    page, dim = 16, 32
    k = torch.zeros(1, 32 + n, 1, dim)
    k[:, 1:32:2, :, 0] = 1.0
    k[:, 32:, :, 0] = 24.0  # the queries' own tokens: weights of exp(-24 scale)
    v = torch.tensor([4.0, 1.0, 1.5, 2.0, 3.0, 6.0, 4.0, 3.0]).repeat(4).expand(1, 32 + n, 1, dim).clone()
    v[:, 1::2] = -torch.tensor([6.0, 1.5, 2.0, 3.0, 4.0, 6.0, 6.0, 4.0]).repeat(4)
    q = torch.zeros(1, n, 2, dim)
    q[..., 0] = -1.0
    cache = mx4_cache(8, 1, page, dim, device=DEV)
    tables = torch.tensor([[5, 2, 7, 1, 0]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([32 + n], dtype=torch.int32, device=DEV)
    mx4_cache_append(cache, k.to(dtype).to(DEV), v.to(dtype).to(DEV), tables, lengths)
    see = torch.arange(32 + n)[None] <= (torch.arange(n) + 32)[:, None]
    for i in range(24):
        scale = float(torch.tensor(0.25 + 0.0171 * i, dtype=torch.float32))
        y = cached_attention_forward(q.to(dtype).to(DEV), cache, tables, lengths, scale=scale)
        ref, mag, _ = ora.attend(q[0, :, 0], k[0, :, 0], v[0, :, 0], see, scale)
        score = 4 * STEP * 24 * scale
        bound = mag * (2.0 ** -16 + 2 * score + 8 * STEP + 4 * (32 + n) * STEP) + half_step(dtype) * ref.abs()
        for h in range(2):
            within(y[0, :, h], ref, bound, f"{dtype} {n} scale {scale} w {math.exp(-scale)}")
