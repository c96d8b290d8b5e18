"""Sequences on the GPU as a server keeps them -- prompts, forks, steps, ends, a compaction -- every step against the oracle."""

import pytest
import torch

from oracle import mx4 as ora
from sparseflow_amd.Kernels.cached_attention import cached_attention_forward, cached_attention_step, mx4_cache, mx4_cache_append
from sparseflow_amd.Kernels.pages import pages_compact, pages_fork, pages_resize
from tests.gpu_helpers import DEV, announce
from tests.mx4_checks import attention_bound, within

pytestmark = pytest.mark.gpu
PAGE, KV, HEADS, DIM = 8, 2, 4, 64


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_every_step_of_a_server(dtype):
    """What each row's tokens are is kept in a list of its own: pages that are shared, copied, given back and moved must
    hold the same."""
    announce(f"serving {dtype}")
    g = torch.Generator().manual_seed(3)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    new = lambda *n: torch.randn(*n, generator=g).to(dtype)  # noqa: E731
    cache = mx4_cache(30, KV, PAGE, DIM, device=DEV)
    for t in cache:
        t.fill_(255)
    refs, lengths = torch.zeros(30, dtype=torch.int32, device=DEV), torch.zeros(6, dtype=torch.int32, device=DEV)
    tables = torch.full((6, 9), -1, dtype=torch.int32, device=DEV)
    lines = {}  # row -> its keys and values, in 64 bits as the format holds them

    def held(t):
        c, s = ora.quantize(t)
        return ora.values(c[..., 0::2] + 16 * c[..., 1::2], s, DIM)

    def check(y, q, rows, counts):
        first = 0
        for r, n in zip(rows, counts):
            k, v = lines[r]
            see = torch.arange(k.shape[0])[None] <= (k.shape[0] - n + torch.arange(n))[:, None]
            for h in range(HEADS):
                ref, mag, big = ora.attend(q[first:first + n, h], k[:, h // 2], v[:, h // 2], see, DIM ** -0.5)
                within(y[first:first + n, h], ref, attention_bound(dtype, DIM, k.shape[0], ref, mag, big), f"row {r} head {h}")
            first += n

    def prompt(rows, counts):
        granted = pages_resize(refs, tables, lengths, ints(*rows), ints(*counts), PAGE, cache)
        assert granted.tolist() == [1] * len(rows)
        k, v, q = new(sum(counts), KV, DIM), new(sum(counts), KV, DIM), new(sum(counts), HEADS, DIM)
        off = ints(0, *torch.tensor(counts).cumsum(0).tolist())
        mx4_cache_append(cache, k.to(DEV), v.to(DEV), tables, lengths, slots=ints(*rows), offsets=off, max_len=max(counts))
        y = cached_attention_forward(q.to(DEV), cache, tables, lengths, slots=ints(*rows), offsets=off, max_len=max(counts))
        for r, kb, vb in zip(rows, held(k).split(counts), held(v).split(counts)):
            lines[r] = (kb, vb)
        check(y, q, rows, counts)

    def step(rows):
        sizes = [lines[r][0].shape[0] + 1 for r in rows]
        granted = pages_resize(refs, tables, lengths, ints(*rows), ints(*sizes), PAGE, cache)
        assert granted.tolist() == [1] * len(rows)
        k, v, q = new(len(rows), KV, DIM), new(len(rows), KV, DIM), new(len(rows), HEADS, DIM)
        mx4_cache_append(cache, k[:, None].to(DEV), v[:, None].to(DEV), tables, lengths, slots=ints(*rows))
        y = cached_attention_step(q.to(DEV), cache, tables, lengths, slots=ints(*rows))
        for i, r in enumerate(rows):
            lines[r] = tuple(torch.cat([a, b[i:i + 1]]) for a, b in zip(lines[r], (held(k), held(v))))
        check(y, q, rows, [1] * len(rows))

    prompt([0, 3], [19, 32])
    assert pages_fork(refs, tables, lengths, ints(0, 0, 3), ints(1, 2, 5), PAGE, cache).tolist() == [1, 1, 1]
    lines.update({1: lines[0], 2: lines[0], 5: lines[3]})
    for _ in range(7):
        step([0, 1, 2, 3, 5])
    assert pages_resize(refs, tables, lengths, ints(0, 3), ints(0, 0), PAGE, cache).tolist() == [1, 1]
    pages_resize(refs, tables, lengths, ints(1), ints(21), PAGE, cache)  # (back to 21 of its 26 tokens)
    lines[1] = tuple(t[:21] for t in lines[1])
    used = int((refs > 0).sum())
    assert pages_compact(refs, tables, cache).tolist() == [used] and not refs[used:].any()
    step([1, 2, 5])
    prompt([4], [40])
    step([4, 2, 1, 5])
    # Every page is as often in use as the tables say.
    there = tables[tables >= 0].long().cpu()
    assert torch.equal(torch.bincount(there, minlength=30), refs.cpu().long())
