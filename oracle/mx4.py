"""Microscaled 4-bit numbers, the Linear over them, attention over a paged cache in the
format, and the pages of a cache, restated in 64 bits and plain Python.

Every function that sums returns, beside its result, what an error bound needs: the
sum of the magnitudes of its terms."""

from __future__ import annotations

import math

import torch

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def quantize(x: torch.Tensor):
    """x [..., dim] -> (codes [..., 32 blocks] one each, scale bytes [..., blocks]) as integers."""
    x = x.double()
    x = torch.nn.functional.pad(x, (0, -x.shape[-1] % 32)).unflatten(-1, (-1, 32))
    rows = x.reshape(-1, 32).tolist()
    codes, scales = [], []
    for row in rows:
        if any(math.isnan(v) or math.isinf(v) for v in row):
            codes.append([0] * 32)
            scales.append(255)
            continue
        top = max(abs(v) for v in row)
        e = max(math.frexp(top)[1] - 1 - 2, -127) if top > 0 else -127
        out = []
        for v in row:
            a = math.ldexp(abs(v), -e)
            near = min(range(8), key=lambda i: (abs(a - LEVELS[i]), i % 2))
            out.append(near + (8 if math.copysign(1.0, v) < 0 else 0))
        codes.append(out)
        scales.append(e + 127)
    lead, n = x.shape[:-2], x.shape[-2]
    return (torch.tensor(codes, dtype=torch.uint8).reshape(*lead, 32 * n), torch.tensor(scales, dtype=torch.uint8).reshape(*lead, n))


def unpack(packed: torch.Tensor) -> torch.Tensor:
    """Two codes to a byte -> one each."""
    return torch.stack([packed % 16, packed // 16], dim=-1).flatten(-2)


def values(packed: torch.Tensor, scales: torch.Tensor, size: int) -> torch.Tensor:
    c = unpack(packed.cpu()).long()
    s = scales.cpu().long()
    v = torch.tensor(LEVELS, dtype=torch.float64)[c % 8] * (1 - 2 * (c // 8))
    f = torch.where(s == 255, torch.full(s.shape, math.nan, dtype=torch.float64), torch.ldexp(torch.ones(s.shape, dtype=torch.float64), s - 127))
    return (v.unflatten(-1, (-1, 32)) * f[..., None]).flatten(-2)[..., :size]


def linear(x: torch.Tensor, w: torch.Tensor, bias=None):
    """(x W^T + bias, sum of the terms' magnitudes), x and w as values."""
    x, w = x.double().cpu(), w.double().cpu()
    b = 0 if bias is None else bias.double().cpu()
    return x @ w.t() + b, x.abs() @ w.abs().t() + (0 if bias is None else b.abs())


def attend(q, k, v, places, scale: float):
    """q [n, dim], k and v [tokens, dim] at `places` (which tokens each query sees: a bool
    [n, tokens]) -> (y, the sum of the weights times |v|, the largest sum of |q k| scale)."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    y, mag, big = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(q.shape[0], dtype=torch.float64)
    for i in range(q.shape[0]):
        see = places[i]
        if not see.any():
            continue
        p = torch.softmax(k[see] @ q[i] * scale, 0)
        y[i], mag[i] = p @ v[see], p @ v[see].abs()
        big[i] = (k[see].abs() @ q[i].abs()).max() * abs(scale)
    return y, mag, big


class Pages:
    """The pages of a cache as plain lists: what each row of tables holds, and what is in a page."""

    def __init__(self, refs, tables, lengths, page, contents):
        self.page, self.width = page, tables.shape[1]
        self.refs = refs.tolist()
        self.lengths = lengths.tolist()
        self.rows = [[int(p) for p in t[: -(-n // page)]] for t, n in zip(tables, self.lengths)]
        self.contents = list(contents)

    def count(self, n):
        return -(-n // self.page)

    def _deal(self, needs):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        out, at = [], 0
        for n in needs:
            out.append(free[at:at + n] if at + n <= len(free) or n == 0 else None)
            at += n
        return out

    def resize(self, rows, sizes):
        granted, grow, named = [0] * len(rows), [], set()
        for i, (r, n) in enumerate(zip(rows, sizes)):
            fine = r not in named and 0 <= r < len(self.rows) and 0 <= n and self.count(n) <= self.width
            named.add(r)
            if not fine:
                continue
            if n > self.lengths[r]:
                grow.append((i, r, n))
                continue
            for p in self.rows[r][self.count(n):]:
                self.refs[p] -= 1
            self.rows[r] = self.rows[r][: self.count(n)]
            self.lengths[r], granted[i] = n, 1
        copies = [self.lengths[r] % self.page != 0 and self.refs[self.rows[r][-1]] > 1 for _, r, _ in grow]
        for (i, r, n), copy, got in zip(grow, copies, self._deal([self.count(n) - len(self.rows[r]) + c
                                                                  for (_, r, n), c in zip(grow, copies)])):
            if got is None:
                continue
            if copy:
                old = self.rows[r].pop()
                self.contents[got[0]] = self.contents[old]
                self.refs[old] -= 1
            for p in got:
                self.refs[p] = 1
            self.rows[r] += got
            self.lengths[r], granted[i] = n, 1
        return granted

    def fork(self, parents, children):
        granted, named, todo = [0] * len(parents), set(), []
        before = [list(r) for r in self.rows], list(self.lengths)
        for i, (a, b) in enumerate(zip(parents, children)):
            fine = b not in named and 0 <= b < len(self.rows) and 0 <= a < len(self.rows) and before[1][b] == 0
            named.add(b)
            todo.append((a, b) if fine else None)
        needs = [int(t is not None and before[1][t[0]] % self.page != 0) for t in todo]
        for i, (t, got) in enumerate(zip(todo, self._deal(needs))):
            if t is None or got is None:
                continue
            pages, n = before[0][t[0]], before[1][t[0]]
            whole = pages[: n // self.page]
            for p in whole:
                self.refs[p] += 1
            for p in got:
                self.refs[p] = 1
                self.contents[p] = self.contents[pages[-1]]
            self.rows[t[1]], self.lengths[t[1]], granted[i] = whole + got, n, 1
        return granted

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if self.refs[p] <= 0]
        strays = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(strays, holes))
        for a, b in to.items():
            self.contents[b], self.refs[b], self.refs[a] = self.contents[a], self.refs[a], 0
        self.rows = [[to.get(p, p) for p in r] for r in self.rows]
        return live

    def tables(self):
        return [r + [-1] * (self.width - len(r)) for r in self.rows]
