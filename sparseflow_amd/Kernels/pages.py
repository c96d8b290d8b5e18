"""The pages of a cache (Kernels/cached_attention.py's, or any tensors [pages, ...]):
sequences grow, shrink, end and fork, and pools are compacted, on the device and without
a synchronisation.

refs int32 [pages]: how many table rows use a page, 0 is free.  Row r of tables, int32
[rows, width], has ceil(lengths[r] / page_size) pages in front and -1 behind.  Rows share
full pages; a page that a row writes to is its own.

A call's requests are dealt with as one: what is freed comes first, then the free pages
go, lowest first, to the requests in turn, until one cannot have what it needs; that one
and those behind it that need pages are refused, and a refused request changes nothing.
Refused too: a row outside tables, a size that is negative or wider than the table, a row
that an earlier request of the call names.  A call on the device takes 2^20 requests at most,
each of which looks through those before it, and a copy 2^24 pairs.  `pools` are the tensors
whose pages have to be copied along.

Device tensors run sf_pages_*; host tensors the torch forms below."""

from __future__ import annotations

from typing import Dict, List, Sequence, Tuple

import torch

from .. import _lib
from ._sequences import Plans, overlap, reaches, signature, surely_apart


def _check_pools(pools: Sequence[torch.Tensor], device: torch.device, pages: int) -> Tuple[torch.Tensor, ...]:
    pools = tuple(pools)
    if len(pools) > _lib.SF_MAX_POOLS:
        raise _lib.UnsupportedError(f"{len(pools)} pools: {_lib.SF_MAX_POOLS} at most")
    for i, t in enumerate(pools):
        if t.dim() < 1 or t.shape[0] != pages or t.device != device or not t.is_contiguous():
            raise ValueError(f"pool {i} is {tuple(t.shape)} on {t.device}: a contiguous ({pages}, ...) on {device} is wanted")
    return pools


def _check_ints(t: torch.Tensor, name: str, device: torch.device, shape: Tuple[int, ...]) -> None:
    if tuple(t.shape) != shape or t.dtype != torch.int32 or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} is {tuple(t.shape)} {t.dtype} on {t.device}: a contiguous {shape} int32 on {device} is "
                         "wanted")


def _check_apart(written: Dict[str, torch.Tensor], read: Dict[str, torch.Tensor]) -> None:
    names = list(written)
    for i, name in enumerate(names):
        for other, t in [(n, written[n]) for n in names[i + 1:]] + list(read.items()):
            if overlap(written[name], t):
                raise ValueError(f"{name} shares memory with {other}")


_plans = Plans()


def _check(refs, tables, lengths, page_size, pools, **requests) -> Tuple[int, Tuple[torch.Tensor, ...]]:
    """-> (page_size, pools) of a call whose arguments fit together and lie apart."""
    page_size, pools = int(page_size), tuple(pools)
    written = (refs, tables, *pools) if lengths is None else (refs, tables, lengths, *pools)
    read = tuple(requests.values())
    key = (signature(*written), signature(*read), page_size, lengths is None)
    spans = _plans.get(key) or _plans.make(key, _check_shapes, refs, tables, lengths, page_size, pools, requests)
    if not surely_apart(written, spans[0], read, spans[1]):
        named = {"refs": refs, "tables": tables, **({} if lengths is None else {"lengths": lengths})}
        _check_apart({**named, **{f"pool {i}": t for i, t in enumerate(pools)}}, requests)
    return page_size, pools


def _check_shapes(refs, tables, lengths, page_size, pools, requests) -> tuple:
    """-> the bytes that what is written, and what is read, reach over."""
    if refs.dim() != 1:
        raise ValueError(f"refs is {tuple(refs.shape)}: (pages,) is wanted")
    _check_ints(refs, "refs", refs.device, tuple(refs.shape))
    if tables.dim() != 2:
        raise ValueError(f"tables is {tuple(tables.shape)}: (rows, width) is wanted")
    _check_ints(tables, "tables", refs.device, tuple(tables.shape))
    if lengths is not None:
        _check_ints(lengths, "lengths", refs.device, (int(tables.shape[0]),))
    if page_size < 1:
        raise ValueError(f"page_size {page_size}: 1 or more is wanted")
    size = None
    for name, t in requests.items():
        if t.dim() != 1 or (size is not None and t.numel() != size):
            raise ValueError(f"{name} is {tuple(t.shape)}: as many as the other requests are wanted")
        size = t.numel()
        _check_ints(t, name, refs.device, (size,))
    _check_pools(pools, refs.device, int(refs.shape[0]))
    return reaches(*((refs, tables) if lengths is None else (refs, tables, lengths)), *pools), reaches(*requests.values())


def _buffers(refs: torch.Tensor, requests: int, results: int) -> Tuple[torch.Tensor, torch.Tensor]:
    return (torch.empty(results, dtype=torch.int32, device=refs.device),
            torch.empty(_lib.pages_workspace_size(refs.numel(), requests), dtype=torch.uint8, device=refs.device))


def _host_deal(refs: torch.Tensor, need: List[int]) -> List[List[int]]:
    """Pages for every request (None: it gets none), the lowest free ones first."""
    free = (refs <= 0).nonzero().flatten().tolist()
    got, at = [], 0
    for n in need:
        n = max(n, 0)
        got.append(free[at:at + n] if at + n <= len(free) else None if n else [])
        at += n
    return got


def _copy_page(pools, source: int, target: int) -> None:
    for pool in pools:
        pool[target] = pool[source]


@torch.no_grad()
def _host_resize(refs, tables, lengths, rows, sizes, page, pools, granted) -> None:
    pages, width = refs.numel(), tables.shape[1]
    up = lambda n: -(-n // page)  # noqa: E731
    seen, todo = set(), []
    for q, (row, size) in enumerate(zip(rows.tolist(), sizes.tolist())):
        ok = row not in seen and 0 <= row < tables.shape[0] and size >= 0 and up(size) <= width
        seen.add(row)
        old = max(0, int(lengths[row])) if ok else 0
        granted[q] = int(ok)
        if ok and size <= old:
            for i in range(up(size), min(up(old), width)):
                p = int(tables[row, i])
                if 0 <= p < pages:
                    refs[p] -= 1
                tables[row, i] = -1
            lengths[row] = size
        elif ok:
            todo.append((q, row, old, size))
    need, shared = [], []
    for _, row, old, size in todo:
        last = int(tables[row, old // page]) if old % page else -1
        shared.append(0 <= last < pages and int(refs[last]) > 1)
        need.append(up(size) - up(old) + shared[-1])
    for (q, row, old, size), copied, got in zip(todo, shared, _host_deal(refs, need)):
        if got is None:
            granted[q] = 0
            continue
        first = up(old) - copied
        if copied:
            last = int(tables[row, first])
            _copy_page(pools, last, got[0])
            refs[last] -= 1
        for i, p in enumerate(got):
            tables[row, first + i] = p
            refs[p] = 1
        lengths[row] = size


@torch.no_grad()
def _host_fork(refs, tables, lengths, parents, children, page, pools, granted) -> None:
    pages, rows, width = refs.numel(), tables.shape[0], tables.shape[1]
    seen, todo, need = set(), [], []
    for q, (parent, child) in enumerate(zip(parents.tolist(), children.tolist())):
        ok = child not in seen and 0 <= child < rows and 0 <= parent < rows and int(lengths[child]) == 0
        seen.add(child)
        n = int(lengths[parent]) if ok else 0
        ok = ok and n >= 0 and -(-n // page) <= width
        todo.append((q, parent, child, n, ok))
        need.append(int(n % page != 0) if ok else 0)
    for (q, parent, child, n, ok), got in zip(todo, _host_deal(refs, need)):
        granted[q] = int(ok and got is not None)
        if not ok or got is None or n == 0:
            continue
        whole = n // page
        for i in range(whole):
            p = int(tables[parent, i])
            tables[child, i] = p
            if 0 <= p < pages:
                refs[p] += 1
        if got:
            last = int(tables[parent, whole])
            tables[child, whole] = got[0]
            refs[got[0]] = 1
            if 0 <= last < pages:
                _copy_page(pools, last, got[0])
        lengths[child] = n


def pages_resize(refs: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, rows: torch.Tensor, sizes: torch.Tensor,
                 page_size: int, pools: Sequence[torch.Tensor] = ()) -> torch.Tensor:
    """Row rows[i] of tables to sizes[i] tokens (int32 both; 0 ends a sequence) -> granted
    int32 [requests].

    A row that shrinks gives its last pages back; one that grows gets new ones, whose
    contents are what they were.  Before it grows, a partial last page that others use too
    is replaced by a copy.
    """
    page_size, pools = _check(refs, tables, lengths, page_size, pools, rows=rows, sizes=sizes)
    if not refs.is_cuda:
        granted = torch.zeros(rows.numel(), dtype=torch.int32)
        _host_resize(refs, tables, lengths, rows, sizes, page_size, pools, granted)
        return granted
    granted, workspace = _buffers(refs, rows.numel(), rows.numel())
    _lib.pages_resize(refs, tables, lengths, rows, sizes, page_size, pools, granted, workspace)
    return granted


def pages_fork(refs: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, parents: torch.Tensor, children: torch.Tensor,
               page_size: int, pools: Sequence[torch.Tensor] = ()) -> torch.Tensor:
    """Row children[i], which is empty (else the request is refused), becomes what row
    parents[i] is before the call -> granted int32 [requests].

    It shares the full pages and has a copy of the last, partial one.
    """
    page_size, pools = _check(refs, tables, lengths, page_size, pools, parents=parents, children=children)
    if not refs.is_cuda:
        granted = torch.zeros(parents.numel(), dtype=torch.int32)
        _host_fork(refs, tables, lengths, parents, children, page_size, pools, granted)
        return granted
    granted, workspace = _buffers(refs, parents.numel(), parents.numel())
    _lib.pages_fork(refs, tables, lengths, parents, children, page_size, pools, granted, workspace)
    return granted


def pages_compact(refs: torch.Tensor, tables: torch.Tensor, pools: Sequence[torch.Tensor] = ()) -> torch.Tensor:
    """The n pages in use become pages 0 to n - 1 -> n, int32 [1].

    Those from n on move, in order, to the free ones below it; tables, refs and the pools'
    contents follow.
    """
    _, pools = _check(refs, tables, None, 1, pools)
    if not refs.is_cuda:
        with torch.no_grad():
            used = refs > 0
            n = int(used.sum())
            at = torch.arange(refs.numel())
            source, target = at[used & (at >= n)], at[~used & (at < n)]
            to = at.clone()
            to[source] = target
            for pool in pools:
                pool[target] = pool[source]
            refs[target] = refs[source]
            refs[source] = 0
            there = (tables >= 0) & (tables < refs.numel())
            tables[there] = to[tables[there].long()].int()
            return torch.tensor([n], dtype=torch.int32)
    live, workspace = _buffers(refs, 0, 1)
    _lib.pages_compact(refs, tables, pools, live, workspace)
    return live


def pages_copy(pools: Sequence[torch.Tensor], sources: torch.Tensor, targets: torch.Tensor) -> None:
    """Page sources[i] of every pool to page targets[i] (int32 both).

    No target is named twice, or is a source too.  A pair outside the pools is left out.
    """
    pools = tuple(pools)
    if not pools:
        raise ValueError("pools is empty")
    if pools[0].dim() < 1:
        raise ValueError("pool 0 has no axis of pages")
    pages, device = int(pools[0].shape[0]), pools[0].device
    _check_pools(pools, device, pages)
    if sources.dim() != 1:
        raise ValueError(f"sources is {tuple(sources.shape)}: (pairs,) is wanted")
    _check_ints(sources, "sources", device, tuple(sources.shape))
    _check_ints(targets, "targets", device, tuple(sources.shape))
    _check_apart({f"pool {i}": t for i, t in enumerate(pools)}, {"sources": sources, "targets": targets})
    if not sources.is_cuda:
        with torch.no_grad():
            for s, t in zip(sources.tolist(), targets.tolist()):
                if 0 <= s < pages and 0 <= t < pages and s != t:
                    _copy_page(pools, s, t)
        return
    _lib.pages_copy(pools, sources, targets)
