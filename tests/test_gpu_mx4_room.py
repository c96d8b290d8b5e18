"""Attention over the 4-bit cache on the GPU: lengths that pass the room of the tables."""

import pytest
import torch

from oracle import mx4 as ora
from sparseflow_amd.Kernels.cached_attention import cached_attention_forward, mx4_cache, mx4_cache_append
from tests.gpu_helpers import DEV, announce
from tests.mx4_checks import attention_bound, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 40, 150])
@pytest.mark.parametrize("page,width", [(8, 3), (16, 5), (1, 7), (64, 33)])
@pytest.mark.parametrize("dim", [64, 160])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_lengths_past_the_tables(dtype, dim, page, width, n):
    """Tokens past a table's width are seen by nobody; what the pool's first rows hold is no number."""
    announce(f"attention past the table {dtype} {dim} {page} {width} {n}")
    g = torch.Generator().manual_seed(page)
    room = page * width
    tables = (torch.randperm(2 * width, generator=g).int() + 1).view(2, width).to(DEV)
    cache = mx4_cache(2 * width + 1, 2, page, dim, device=DEV)
    for t in cache:
        t.fill_(255)  # page 0, which is in no table, too
    full = torch.tensor([room, room], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(2, room, 2, dim, generator=g).to(dtype) for _ in "kv")
    mx4_cache_append(cache, k.to(DEV), v.to(DEV), tables, full)
    q = torch.randn(2, n, 4, dim, generator=g).to(dtype)
    for over in ((0, 1), (5, n // 2), (n + 3, 1000)):
        lengths = torch.tensor([room + o for o in over], dtype=torch.int32, device=DEV)
        y = cached_attention_forward(q.to(DEV), cache, tables, lengths).cpu()
        for b in range(2):
            place = room + over[b] - n + torch.arange(n)
            see = torch.arange(room)[None] <= place[:, None]
            for h in range(4):
                held = []
                for codes, scales in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)):
                    rows = tables[b].long()
                    held.append(ora.values(codes[rows, h // 2].flatten(0, 1), scales[rows, h // 2].flatten(0, 1), dim))
                ref, mag, big = ora.attend(q[b, :, h], *held, see, dim ** -0.5)
                within(y[b, :, h], ref, attention_bound(dtype, dim, room, ref, mag, big), f"{over} {b} {h}")
