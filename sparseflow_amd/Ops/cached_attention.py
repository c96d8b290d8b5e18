"""CachedAttention: causal softmax attention of token sequences over a paged 4-bit
cache of their keys and values (Kernels/cached_attention.py, Kernels/pages.py).

Stateful like the neurons (neuron.py) and the scan: a forward continues each sequence
of the batch from where the last one left it, a prompt or a token at a time, until
reset().  Tokens take pages as they come; the sequences of a search share the pages of
what they have in common (select).  Every query sees keys and values in the format, the
call's own tokens included, so a prompt and its tokens one by one agree.  Inference
only."""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from .. import _lib
from ..Kernels._sequences import check_input, check_like
from ..Kernels.cached_attention import MAX_HEAD_DIM, MAX_PAGE, MX4Cache, cached_attention_forward, check_scale, mx4_cache, \
    mx4_cache_append
from ..Kernels.mx4 import blocks_of
from ..Kernels.pages import pages_compact, pages_fork, pages_resize
from ._runtime import host_parents


class _Sequences:
    """A batch's cache: rows 0 to batch - 1 or batch to 2 batch - 1 of the tables are its
    sequences (`slots`), the others are empty: what select() fills."""

    def __init__(self, batch: int, kv_heads: int, head_dim: int, page: int, device: torch.device):
        ints = dict(dtype=torch.int32, device=device)
        self.batch, self.page, self.tokens = batch, page, 0
        # How many pages may be in use at most, by the tokens taken; the device deals them out.
        self.used = 0
        self.cache = mx4_cache(0, kv_heads, page, head_dim, device)
        self.refs = torch.zeros(0, **ints)
        self.tables = torch.full((2 * batch, 0), -1, **ints)
        self.lengths = torch.zeros(2 * batch, **ints)
        self.halves = torch.arange(batch, **ints), torch.arange(batch, 2 * batch, **ints)
        self.slots = self.halves[0]

    def fits(self, batch: int, kv_heads: int, head_dim: int, device: torch.device) -> bool:
        return (self.batch == batch and self.refs.device == device and self.cache.k.shape[1] == kv_heads
                and self.cache.k_scales.shape[3] == blocks_of(head_dim))

    def _pages(self, wanted: int) -> None:
        """The pools hold `wanted` pages at least: those that they have keep their numbers."""
        have = self.refs.numel()
        if wanted <= have:
            return
        more = max(wanted, 2 * have) - have
        longer = lambda t: torch.cat([t, t.new_zeros(more, *t.shape[1:])])  # noqa: E731
        self.cache, self.refs = MX4Cache(*map(longer, self.cache)), longer(self.refs)

    def take(self, tokens: int) -> None:
        """Places for so many more tokens of every sequence."""
        total = self.tokens + tokens
        width = -(-total // self.page)
        self.used += self.batch * (width - -(-self.tokens // self.page))
        if width > self.tables.shape[1]:
            more = max(width, 2 * self.tables.shape[1]) - self.tables.shape[1]
            self.tables = torch.cat([self.tables, self.tables.new_full((2 * self.batch, more), -1)], 1)
        self._pages(self.used)
        pages_resize(self.refs, self.tables, self.lengths, self.slots, torch.full_like(self.slots, total), self.page,
                     self.cache)
        self.tokens = total

    def select(self, parents: torch.Tensor) -> None:
        self._pages(self.used + self.batch)  # (the copies of partial pages, before what they replace ends)
        rest = self.halves[self.slots is self.halves[0]]
        pages_fork(self.refs, self.tables, self.lengths, self.slots[parents.to(self.refs.device)], rest, self.page, self.cache)
        pages_resize(self.refs, self.tables, self.lengths, self.slots, torch.zeros_like(self.slots), self.page)
        self.slots = rest

    def compact(self) -> None:
        self.used = n = int(pages_compact(self.refs, self.tables, self.cache))
        self.cache, self.refs = MX4Cache(*(t[:n].clone() for t in self.cache)), self.refs[:n].clone()


class CachedAttention(nn.Module):
    """q [batch, tokens, heads, head_dim], k and v [batch, tokens, kv_heads, head_dim] -> y like q."""

    def __init__(self, page_size: int = 64, scale: Optional[float] = None):
        super().__init__()
        self.page_size, self.scale = int(page_size), scale
        if not 1 <= self.page_size <= MAX_PAGE or self.page_size & (self.page_size - 1):
            raise ValueError(f"page_size={page_size}: a power of two up to {MAX_PAGE} is wanted")
        if scale is not None:
            check_scale(float(scale))
        self.state: Optional[_Sequences] = None

    def reset(self):
        self.state = None

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        # (Everything is checked before the sequences take the tokens.)
        if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
            raise ValueError(f"q is {tuple(q.shape)}, k {tuple(k.shape)}: (batch, tokens, heads, head_dim) each are wanted, "
                             "alike but for the heads")
        batch, tokens, kv_heads, dim = (int(n) for n in k.shape)
        if kv_heads < 1 or dim < 1 or q.shape[2] < 1 or q.shape[2] % kv_heads:
            raise ValueError(f"q has {q.shape[2]} heads of {dim}: a multiple of k's {kv_heads} is wanted")
        if dim > MAX_HEAD_DIM:
            raise _lib.UnsupportedError(f"head_dim {dim} is over {MAX_HEAD_DIM}")
        check_input(q, "q")
        check_like(k, q, "k", tuple(k.shape))
        check_like(v, q, "v", tuple(k.shape))
        s = self.state
        if s is None or not s.fits(batch, kv_heads, dim, k.device):
            s = self.state = _Sequences(batch, kv_heads, dim, self.page_size, k.device)
        if batch == 0 or tokens == 0:
            return torch.empty_like(q)
        s.take(tokens)
        mx4_cache_append(s.cache, k, v, s.tables, s.lengths, slots=s.slots)
        return cached_attention_forward(q, s.cache, s.tables, s.lengths, slots=s.slots, scale=self.scale)

    def select(self, parents: torch.Tensor) -> None:
        """Sequence i becomes what sequence parents[i] was (integers [batch], checked on the
        host): full pages are shared, partial ones copied."""
        if self.state is not None:
            self.state.select(host_parents(parents, self.state.batch))

    def compact(self) -> None:
        """Gives back the memory of pages that no sequence uses (waits for the device)."""
        if self.state is not None:
            self.state.compact()

    def extra_repr(self) -> str:
        return f"page_size={self.page_size}, scale={self.scale}"
