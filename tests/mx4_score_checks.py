"""A check of attention's rows whose scores are all -infinity, for a device or the host."""

import math

import torch

from sparseflow_amd.Kernels.cached_attention import cached_attention_forward, mx4_cache, mx4_cache_append


def check_scores_of_minus_infinity(dev, dtype, n, old):
    """The softmax of such scores is 0 / 0.  A finite score beside them takes all the weight, and a row that sees no token
    is zeros whatever its query is."""
    g = torch.Generator().manual_seed(n + old)
    page, dim, total = 16, 64, old + n
    width = -(-total // page)
    tables = torch.stack([torch.randperm(width, generator=g), torch.randperm(width, generator=g) + width]).int().to(dev)
    lengths = torch.tensor([total, total], dtype=torch.int32, device=dev)
    cache = mx4_cache(2 * width, 1, page, dim, device=dev)
    k = torch.rand(2, total, 1, dim, generator=g) + 1.0  # between 1 and 2: no code is 0
    v = torch.randn(2, total, 1, dim, generator=g)
    last = old // 2
    k[1, last, 0, 0] = 0.0  # (one finite score of sequence 1: 0 times a finite query)
    mx4_cache_append(cache, k.to(dtype).to(dev), v.to(dtype).to(dev), tables, lengths)
    q = torch.randn(2, n, 2, dim, generator=g)
    q[0, :, :, 7] = -math.inf
    big = torch.finfo(dtype).max if dtype != torch.float16 else math.inf
    q[1] = 0.0
    q[1, :, :, 0] = -big  # (float32 and bf16: every score but one passes float32)
    q = q.to(dtype).to(dev)
    y = cached_attention_forward(q, cache, tables, lengths, scale=1.0 if dtype == torch.float16 else 8.0)
    assert torch.isnan(y[0]).all()
    if dtype != torch.float16:
        want = _value(cache, tables, last, page, dim)
        assert torch.equal(y[1].cpu(), want.to(dtype).expand(n, 2, dim))
    # Fewer tokens than queries: the first rows see none.
    few = n // 2
    y = cached_attention_forward(q, cache, tables, torch.full_like(lengths, few))
    assert not y[:, :n - few].any() and torch.isnan(y[0, n - few:]).all()
    none = cached_attention_forward(q, cache, torch.full_like(tables, -1), lengths)
    assert not none.any()


def _value(cache, tables, t, page, dim):
    from sparseflow_amd.Kernels.mx4 import mx4_dequantize

    p = int(tables[1, t // page])
    return mx4_dequantize(cache.v[p, 0, t % page].clone(), cache.v_scales[p, 0, t % page].clone(), size=dim).cpu()
