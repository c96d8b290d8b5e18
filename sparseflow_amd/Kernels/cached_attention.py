"""Softmax attention over a paged cache of keys and values in the microscaled 4-bit
format (Kernels/mx4.py):

    y_i = sum_t softmax_t(scale q_i . k_t) v_t    over the tokens t up to the query's own

An `MX4Cache` is four tensors [pages, kv_heads, page_size, ...].  Token t of table row r
lies in page tables[r, t // page_size] (int32 [rows, width]; an entry outside the pages
is no page: nothing is written there, and nobody sees its tokens); lengths int32 [rows]
are the tokens of each row, the new ones of a call included: they are the last.  A call's
sequences come dense, [batch, tokens, heads, head_dim], or packed, [total, heads,
head_dim] with `offsets`, and have the table rows `slots` (without: row b), as in the
other entry points of token sequences.  heads / kv_heads query heads in a row share keys
and values.  `Kernels/pages.py` deals pages out.

Device tensors run sf_mx4_cache_append / sf_mx4_attention; host tensors the torch forms
below.  Softmax statistics and sums are float32.  Inference only:
nothing is recorded for a backward pass."""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import _lib
from ._sequences import Plans, check_apart, check_index, check_input, check_like, check_out, host_slots, host_spans, \
    last_contiguous, reaches, signature, surely_apart
from .mx4 import blocks_of, host_dequantize, host_quantize

_appends, _attentions = Plans(), Plans()

MAX_HEAD_DIM = 256
MAX_PAGE = 4096


class MX4Cache(NamedTuple):
    k: torch.Tensor         # uint8 [pages, kv_heads, page_size, 16 blocks of head_dim]
    k_scales: torch.Tensor  # uint8 [pages, kv_heads, page_size, blocks]
    v: torch.Tensor
    v_scales: torch.Tensor


def mx4_cache(pages: int, kv_heads: int, page_size: int, head_dim: int, device=None) -> MX4Cache:
    """An empty cache (zeros)."""
    n = blocks_of(int(head_dim))
    return MX4Cache(*(torch.zeros(pages, kv_heads, page_size, w, dtype=torch.uint8, device=device)
                      for w in (16 * n, n, 16 * n, n)))


def _check_cache(cache, x: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, slots, batch: int, head_dim: int) -> tuple:
    """-> (pages, kv_heads, page_size, rows, width)."""
    if len(cache) != 4 or cache[0].dim() != 4:
        raise ValueError("cache: an MX4Cache is wanted")
    pages, heads, page, _ = (int(v) for v in cache[0].shape)
    n = blocks_of(head_dim)
    for t, name, width in zip(cache, MX4Cache._fields, (16 * n, n, 16 * n, n)):
        if tuple(t.shape) != (pages, heads, page, width) or t.dtype != torch.uint8 or t.device != x.device \
                or not t.is_contiguous():
            raise ValueError(f"cache.{name} is {tuple(t.shape)} {t.dtype} on {t.device}: a contiguous "
                             f"{(pages, heads, page, width)} uint8 on {x.device} is wanted")
    if heads < 1:
        raise ValueError("cache: one head at least is wanted")
    if tables.dim() != 2 or tables.dtype != torch.int32 or tables.device != x.device or not tables.is_contiguous():
        raise ValueError(f"tables is {tuple(tables.shape)} {tables.dtype} on {tables.device}: a contiguous (rows, width) "
                         f"int32 on {x.device} is wanted")
    rows, width = (int(v) for v in tables.shape)
    check_index(lengths, x, "lengths", rows)
    check_index(slots, x, "slots", batch)
    if slots is None and rows != batch:
        raise ValueError(f"tables has {rows} rows: {batch}, or slots, are wanted")
    if head_dim > MAX_HEAD_DIM:
        raise _lib.UnsupportedError(f"head_dim {head_dim} is over {MAX_HEAD_DIM}")
    if page < 1 or page > MAX_PAGE or page & (page - 1):
        raise _lib.UnsupportedError(f"pages of {page} tokens: a power of two up to {MAX_PAGE} is wanted")
    return pages, heads, page, rows, width


def _check_aligned(cache) -> None:
    if cache[0].is_cuda and (cache[0].data_ptr() % 16 or cache[2].data_ptr() % 16):
        raise ValueError("cache: codes that begin at a multiple of 16 bytes are wanted")


def _axes(x: torch.Tensor, name: str, offsets) -> tuple:
    """-> (batch, tokens)."""
    if x.dim() != (4 if offsets is None else 3):
        raise ValueError(f"{name} is {tuple(x.shape)}: (batch, tokens, heads, head_dim), or (total, heads, head_dim) with "
                         "offsets, is wanted")
    check_input(x, name)
    if x.shape[-1] < 1 or x.shape[-2] < 1:
        raise ValueError(f"{name} is {tuple(x.shape)}: a head and a column at least are wanted")
    if offsets is not None and offsets.numel() < 1:
        raise ValueError("offsets is empty: one more than the sequences is wanted")
    batch = int(x.shape[0]) if offsets is None else int(offsets.numel()) - 1
    check_index(offsets, x, "offsets", batch + 1)
    return batch, int(x.shape[-3])


def _strides(x: torch.Tensor) -> tuple:
    return tuple(x.stride()[:3]) if x.dim() == 4 else (0,) + tuple(x.stride()[:2])


def _places(n: int, length: int, table: torch.Tensor, page: int, pages: int):
    """Host: of the last n of `length` tokens, those that have a place: (which, page, row of it)."""
    t = torch.arange(length - n, length)
    i = torch.arange(n)
    fits = (t >= 0) & (t < table.numel() * page)
    t, i = t[fits], i[fits]
    p = table[t // page].long()
    there = (p >= 0) & (p < pages)
    return i[there], p[there], (t % page)[there]


def mx4_cache_append(cache: MX4Cache, k: torch.Tensor, v: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor,
                     slots: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None,
                     max_len: Optional[int] = None) -> None:
    """Quantises the new tokens' keys and values, [batch, tokens, kv_heads, head_dim] or
    packed, into their pages: the last places of each sequence's `lengths` tokens.

    max_len, the longest sequence, sizes the launch of a packed call (default: all its
    tokens).  No two tokens of a call have one place, and the cache shares no memory
    with k and v.
    """
    if k.is_cuda and k.dim() > 0:
        k, v = last_contiguous(k), last_contiguous(v)
    if max_len is not None:
        max_len = int(max_len)
    key = (signature(*cache, k, v, tables, lengths, slots, offsets), max_len)
    plan = _appends.get(key) or _appends.make(key, _check_append, cache, k, v, tables, lengths, slots, offsets, max_len)
    desc, page, pages, written, read = plan
    if not surely_apart(cache, written, (k, v, tables, lengths, slots, offsets), read):
        for i, (t, name) in enumerate(zip(cache, MX4Cache._fields)):
            check_apart(t, "cache." + name, {"k": k, "v": v, "tables": tables, "lengths": lengths, "slots": slots,
                                             "offsets": offsets, **dict(zip(MX4Cache._fields[i + 1:], cache[i + 1:]))})
    if not k.is_cuda:
        with torch.no_grad():
            ks, vs = host_spans(k, offsets), host_spans(v, offsets)
            for s, kb, vb in zip(host_slots(len(ks), tables.shape[0], slots), ks, vs):
                if s < 0:
                    continue
                i, p, r = _places(kb.shape[0], int(lengths[s]), tables[s], page, pages)
                for x, codes, scales in ((kb, cache[0], cache[1]), (vb, cache[2], cache[3])):
                    c, e = host_quantize(x[i])
                    codes[p, :, r] = c
                    scales[p, :, r] = e
        return
    _check_aligned(cache)
    _lib.mx4_cache_append(desc, cache, tables, lengths, k, v, offsets, slots)


def _check_append(cache, k, v, tables, lengths, slots, offsets, max_len):
    """-> (the descriptor of a device call, page_size, pages, bytes that the cache and what is read reach over)."""
    batch, tokens = _axes(k, "k", offsets)
    check_like(v, k, "v", tuple(k.shape))
    dim = int(k.shape[-1])
    pages, heads, page, rows, width = _check_cache(cache, k, tables, lengths, slots, batch, dim)
    if heads != k.shape[-2]:
        raise ValueError(f"k has {k.shape[-2]} heads: the cache's {heads} are wanted")
    spans = reaches(*cache), reaches(k, v, tables, lengths, slots, offsets)
    if not k.is_cuda:
        return (None, page, pages) + spans
    longest = tokens if offsets is None or max_len is None else min(max(max_len, 0), tokens)
    zero = (0, 0, 0)
    return (_lib.mx4_cache_desc(batch, tokens, longest, rows, width, pages, zero, _strides(k), _strides(v), zero, heads, heads,
                               dim, page, k.dtype, 1.0), page, pages) + spans


@torch.no_grad()
def _host_attend(q, cache, length: int, table: torch.Tensor, scale: float) -> torch.Tensor:
    """q [n, heads, dim], a sequence's last tokens -> the same, float32."""
    n, heads, dim = q.shape
    pages, kv, page, _ = cache[0].shape
    y = torch.zeros(n, heads, dim)
    room = min(max(length, 0), table.numel() * page)
    i, p, r = _places(room, room, table, page, pages)
    if n == 0 or i.numel() == 0:
        return y
    place = length - n + torch.arange(n)
    see = i[None] <= place[:, None]
    for h in range(heads):
        g = h // (heads // kv)
        k = host_dequantize(cache[0][p, g, r], cache[1][p, g, r], dim)
        v = host_dequantize(cache[2][p, g, r], cache[3][p, g, r], dim)
        w = (q[:, h].float() @ k.t() * scale).masked_fill(~see, -float("inf"))
        w = torch.exp(w - torch.clamp(w.amax(-1, keepdim=True), min=-3e38)).masked_fill(~see, 0.0)
        total = w.sum(-1, keepdim=True)
        out = w @ v
        bad = ~torch.isfinite(v).all(-1)
        if bad.any():  # 0 times such a value is no 0: each row takes those that it sees
            for j in range(n):
                out[j] = w[j, see[j]] @ v[see[j]]
        y[:, h] = torch.where(see.any(-1, keepdim=True), out / total, torch.zeros(()))
    return y


def check_scale(scale: float) -> float:
    """(NaN is below nothing; times log2(e) it has to be a float32.)"""
    if not abs(scale) < 2.0 ** 127:
        raise ValueError(f"scale is {scale}: a number below 2^127 is wanted")
    return scale


def cached_attention_forward(q: torch.Tensor, cache: MX4Cache, tables: torch.Tensor, lengths: torch.Tensor,
                             slots: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None,
                             max_len: Optional[int] = None, scale: Optional[float] = None,
                             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q [batch, tokens, heads, head_dim], or [total, heads, head_dim] with offsets -> y like q.

    The queries are each sequence's last tokens, whose keys and values the cache holds
    (mx4_cache_append): query i of n has place lengths[slot] - n + i and sees the tokens up
    to it.  One that sees none (an empty sequence, a place before the first, a slot
    outside tables, no page): zeros.  scale: head_dim ** -0.5 by default, a number below 2^127;
    scores that are all -infinity, or that hold a NaN or +infinity, give NaN.  out may be q;
    apart from that it shares no memory with what is read.  Rows of a packed q that are no
    sequence's are left as they are in out.
    """
    return _attention(q, cache, tables, lengths, slots, offsets, max_len, scale, out)


def cached_attention_step(q: torch.Tensor, cache: MX4Cache, tables: torch.Tensor, lengths: torch.Tensor,
                          slots: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of each sequence: q [batch, heads, head_dim] -> y like q
    (cached_attention_forward with one query a sequence)."""
    if q.dim() != 3:
        raise ValueError(f"q is {tuple(q.shape)}: (batch, heads, head_dim) is wanted")
    y = _attention(q[:, None], cache, tables, lengths, slots, None, None, scale, None if out is None else out[:, None])
    return y[:, 0] if out is None else out


def _attention(q, cache, tables, lengths, slots, offsets, max_len, scale, out):
    if q.is_cuda and q.dim() > 0:
        q = last_contiguous(q)
    if max_len is not None:
        max_len = int(max_len)
    scale = float(q.shape[-1]) ** -0.5 if scale is None and q.dim() > 0 and q.shape[-1] > 0 else float(scale or 0.0)
    check_scale(scale)
    key = (signature(q, *cache, tables, lengths, slots, offsets, out), max_len, scale)
    desc, = _attentions.get(key) or _attentions.make(key, _check_attention, q, cache, tables, lengths, slots, offsets,
                                                     max_len, scale, out)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    else:
        check_apart(out, "out", {"q": q, **dict(zip(MX4Cache._fields, cache)), "tables": tables, "lengths": lengths,
                                  "slots": slots, "offsets": offsets},
                    same=("q",))
    if not q.is_cuda:
        spans = host_spans(q, offsets)
        for s, qb, yb in zip(host_slots(len(spans), tables.shape[0], slots), spans, host_spans(out, offsets)):
            yb.copy_(_host_attend(qb, cache, int(lengths[s]), tables[s], scale) if s >= 0 else torch.zeros(qb.shape))
        return out
    _check_aligned(cache)
    workspace = torch.empty(desc[2], dtype=torch.uint8, device=q.device) if desc[2] else None
    _lib.mx4_attention(desc, cache, tables, lengths, q, offsets, slots, out, workspace)
    return out


def _check_attention(q, cache, tables, lengths, slots, offsets, max_len, scale, out):
    """-> (the descriptor of a device call,)."""
    batch, tokens = _axes(q, "q", offsets)
    heads, dim = int(q.shape[-2]), int(q.shape[-1])
    pages, kv, page, rows, width = _check_cache(cache, q, tables, lengths, slots, batch, dim)
    if heads % kv:
        raise ValueError(f"q has {heads} heads: a multiple of the cache's {kv} is wanted")
    if out is not None:
        check_like(out, q, "out", tuple(q.shape))
        check_out(out, "out")
        if out.stride(-1) != 1 and dim > 1:
            raise ValueError("out: a contiguous last axis is wanted")
    if not q.is_cuda:
        return (None,)
    longest = tokens if offsets is None or max_len is None else min(max(max_len, 0), tokens)
    # (A new out has the default strides.)
    y = torch.empty(q.shape, device="meta") if out is None else out
    zero = (0, 0, 0)
    return (_lib.mx4_cache_desc(batch, tokens, longest, rows, width, pages, _strides(q), zero, zero, _strides(y), heads, kv,
                                dim, page, q.dtype, scale),)
