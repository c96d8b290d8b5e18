"""The 4-bit operators as a user of this package calls them: microscaled 4-bit
quantisation and the Linear over such weights, attention over a paged cache held
in that format, and the handling of the cache's pages.

Every case is a plain dict; `op` selects the path:

  quant    Kernels.mx4.mx4_quantize, then mx4_dequantize of what it gave
  linear   Kernels.mx4.mx4_linear_forward on float rows
  linear4  mx4_quantize of the rows, then mx4_linear_forward on them
  attend   Kernels.cached_attention.mx4_cache_append, then cached_attention_forward
           (new tokens of each sequence), or cached_attention_step (one of each)
  fork     Kernels.pages.pages_fork of the sequences that go on, pages_resize of those that ended
  compact  pages_resize of the sequences that ended, pages_compact, pages_resize of new ones

`own` chooses between those and the operators' plain forms in torch.

Format: blocks of 32 along the last axis, one byte 127 + e each (255: not a number);
values +-{0, .5, 1, 1.5, 2, 3, 4, 6} 2^e as 4-bit codes (sign, then the index), two to a
byte with the first in the low half; rows padded with code 0 to whole blocks.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quant(rows, dim, dtype):
    return {"op": "quant", "rows": rows, "dim": dim, "dtype": dtype}


def _linear(rows, inputs, outputs, dtype, four=False, bias=False):
    return {"op": "linear4" if four else "linear", "rows": rows, "inputs": inputs, "outputs": outputs, "dtype": dtype,
            "bias": bias}


def _attend(batch, tokens, before, heads, kv_heads, head_dim, page, dtype, packed=False, step=False):
    return {"op": "attend", "batch": batch, "tokens": tokens, "before": before, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "dtype": dtype, "packed": packed, "step": step}


def _pages(op, rows, length, kv_heads, head_dim, page):
    return {"op": op, "rows": rows, "length": length, "kv_heads": kv_heads, "head_dim": head_dim, "page": page}


def listed():
    return [
        # One image's tokens of float32, an odd width: latency.
        dict(_quant(196, 1037, "f32"), name="quant_small"),
        # The activations of a long prompt before a wide projection.
        dict(_quant(32768, 8192, "bf16"), name="quant_large"),
        # A short prompt in float32 through a projection of odd sizes: latency.
        dict(_linear(37, 1000, 1037, "f32", bias=True), name="linear_small"),
        # One new token through a wide projection.
        dict(_linear(1, 4096, 12288, "bf16"), name="linear_token"),
        # The prompts of a batch, activations in 16 bits: the largest case.
        dict(_linear(8192, 4096, 16384, "bf16"), name="linear_prompt"),
        # The same with activations (or spikes) in 4 bits too.
        dict(_linear(8192, 4096, 16384, "bf16", four=True), name="linear4_prompt"),
        # One new token of one sequence far into a long document, small pages.
        dict(_attend(1, 1, 100000, 64, 8, 128, 16, "f16", step=True), name="attend_document"),
        # One new token of each of 64 sequences of a serving batch, of lengths from none to 16384.
        dict(_attend(64, 1, 16384, 32, 8, 128, 64, "bf16", step=True, packed=True), name="attend_batch"),
        # Prompts of a serving batch, packed without padding, some continuing what was read before.
        dict(_attend(13, 700, 1500, 20, 5, 80, 32, "f16", packed=True), name="attend_packed"),
        # Two long prompts.
        dict(_attend(2, 8192, 0, 32, 8, 128, 64, "bf16"), name="attend_prompt"),
        # A step of a beam search: 256 beams go on from half of the 256 before them.
        dict(_pages("fork", 256, 3000, 8, 128, 64), name="pages_fork"),
        # Half of the sequences of a pool have ended: the others move together, new ones come in.
        dict(_pages("compact", 128, 8000, 8, 128, 64), name="pages_compact"),
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread over their logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case; a third of the widths are no multiple of anything."""
    op = rng.choice(["quant", "linear", "linear", "linear", "linear4", "step", "step", "attend", "attend", "fork", "compact"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    odd = rng.random() < 0.33
    while True:
        if op == "quant":
            rows, dim = _log(rng, 1, 40000), _log(rng, 33, 9000)
            dim = dim if odd else -(-dim // 64) * 64
            if rows * dim > 2 ** 28:
                continue
            return _quant(rows, dim, dtype)
        if op in ("linear", "linear4"):
            rows, inputs, outputs = _log(rng, 1, 8192), _log(rng, 64, 9000), _log(rng, 64, 17000)
            if not odd:
                inputs, outputs = -(-inputs // 128) * 128, -(-outputs // 128) * 128
            if rows * inputs * outputs > 2 ** 39 // (6 if dtype == "f32" else 2 if dtype == "f16" else 1):
                continue
            return _linear(rows, inputs, outputs, dtype, op == "linear4", rng.random() < 0.5)
        if op in ("step", "attend"):
            kv = rng.choice([1, 2, 4, 8])
            heads = kv * rng.choice([1, 2, 4, 7, 8, 16])
            dim = rng.randint(20, 200) if odd else rng.choice([64, 64, 128, 128, 256])
            page = rng.choice([8, 16, 32, 64, 64, 256])
            batch, before = _log(rng, 1, 64), _log(rng, 1, 30000) if rng.random() < 0.8 else 0
            packed = rng.random() < 0.6
            if op == "step":
                if batch * before * kv * (dim + 31) > 2 ** 30:
                    continue
                return _attend(batch, 1, before, heads, kv, dim, page, dtype, packed, True)
            tokens = _log(rng, 1, 8192)
            if batch * tokens * (tokens + before) * heads * max(dim, 64) > 2 ** 38 // (4 if dtype == "f32" else 2 if dtype == "f16" else 1):
                continue
            if batch * (tokens + before) * kv * (dim + 31) > 2 ** 30:
                continue
            return _attend(batch, tokens, before, heads, kv, dim, page, dtype, packed)
        rows, length, kv = 2 * _log(rng, 1, 128), _log(rng, 40, 8000), rng.choice([1, 4, 8])
        if rows * length * kv > 2 ** 23:
            continue
        return _pages(op, rows, length, kv, rng.choice([64, 128]), rng.choice([16, 32, 64]))


def _lengths(case):
    """(new tokens, tokens before) of every sequence; packed: the first has all of the case's, others from none."""
    b, n, before = case["batch"], case["tokens"], case["before"]
    if not case["packed"]:
        return [n] * b, [before] * b
    g = torch.Generator().manual_seed(b * 100003 + n * 17 + before)
    low = 1 if case["step"] else 0
    new = [int(v) for v in torch.randint(low, n + 1, (b,), generator=g)]
    old = [int(v) for v in torch.randint(0, before + 1, (b,), generator=g)]
    new[0], old[0] = n, before
    return new, old


def _page_lengths(case):
    g = torch.Generator().manual_seed(case["rows"] * 100003 + case["length"])
    return [int(v) for v in torch.randint(case["length"] // 2, case["length"] + 1, (case["rows"],), generator=g)]


def _full(n, page):
    return -(-n // page)


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(seed)
    op = case["op"]

    def randn(*shape, dtype=torch.float32, gain=1.0):
        return (torch.randn(shape, generator=g, device=dev) * gain).to(dtype)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    s = {"case": dict(case)}
    if op == "quant":
        s["x"] = randn(case["rows"], case["dim"], dtype=DTYPES[case["dtype"]])
    elif op in ("linear", "linear4"):
        s["x"] = randn(case["rows"], case["inputs"], dtype=DTYPES[case["dtype"]])
        s["weight"] = _quantized(randn(case["outputs"], case["inputs"], gain=case["inputs"] ** -0.5))
        s["bias"] = randn(case["outputs"], gain=0.2) if case["bias"] else None
    elif op == "attend":
        dt, kv, dim, page = DTYPES[case["dtype"]], case["kv_heads"], case["head_dim"], case["page"]
        new, old = _lengths(case)
        total = [a + b for a, b in zip(new, old)]
        width = max(1, _full(max(total), page))
        used = sum(_full(n, page) for n in total)
        pages = used + 3
        order = torch.randperm(pages, generator=g, device=dev)[:used].to(torch.int32)
        s["tables"] = torch.full((case["batch"], width), -1, dtype=torch.int32, device=dev)
        at = torch.arange(width, device=dev)[None] < ints([_full(n, page) for n in total])[:, None]
        s["tables"][at] = order
        s["lengths"], s["max_len"] = ints(total), max(new)
        cache = []
        for _ in "kv":  # what was read before, whole pages of it
            codes, scales = _quantized(randn(pages, kv, page, dim))
            cache += [codes, scales]
        s["cache"] = cache
        off = [0]
        for n in new:
            off.append(off[-1] + n)
        s["offsets"] = ints(off) if case["packed"] and not case["step"] else None
        lead = (case["batch"],) if case["step"] else (off[-1],) if case["packed"] else (case["batch"], case["tokens"])
        # The three are views of one projection's output.
        qkv = randn(*lead, case["heads"] + 2 * kv, dim, dtype=dt)
        s["q"], s["k"], s["v"] = qkv.split([case["heads"], kv, kv], dim=-2)
    else:
        rows, kv, dim, page = case["rows"], case["kv_heads"], case["head_dim"], case["page"]
        lens = _page_lengths(case)
        held = [_full(n, page) for n in lens]
        pages = sum(held) + (2 * rows if op == "fork" else 16)
        # Fork: as many rows again, empty, for those that go on.
        s["lengths"] = ints(lens + ([0] * rows if op == "fork" else []))
        s["tables"] = torch.full((s["lengths"].numel(), _full(case["length"], page)), -1, dtype=torch.int32, device=dev)
        order = torch.randperm(pages, generator=g, device=dev)[: sum(held)].to(torch.int32)
        at = torch.arange(s["tables"].shape[1], device=dev)[None] < ints(held)[:, None]
        s["tables"][:rows][at] = order
        s["refs"] = torch.zeros(pages, dtype=torch.int32, device=dev)
        s["refs"][order.long()] = 1
        nb = _full(dim, 32)
        s["pools"] = [torch.randint(0, 256, (pages, kv, page, n), generator=g, device=dev, dtype=torch.uint8)
                      for n in (16 * nb, nb, 16 * nb, nb)]
        if op == "fork":
            s["rows"] = [ints(range(rows)), ints(range(rows, 2 * rows))]
            # Which of a step's beams each beam of the next continues: half of them, some several times.
            s["picks"] = torch.randint(0, max(1, rows // 2), (rows,), generator=g, device=dev) * 2
            s["none"] = ints([0] * rows)
        else:
            half = [list(range(0, rows, 2)), list(range(1, rows, 2))]
            s["rows"] = [ints(h) for h in half]
            s["sizes"] = [ints([lens[r] for r in h]) for h in half]
            s["none"] = [ints([0] * len(h)) for h in half]
    return s


# ---- plain forms: 32 bits, rounded once at the end ---------------------------


def _padded(x):
    """x with its last axis padded to whole blocks: [..., blocks, 32]."""
    n = -x.shape[-1] % 32
    if n:
        x = torch.cat([x, x.new_zeros(x.shape[:-1] + (n,))], dim=-1)
    return x.unflatten(-1, (-1, 32))


def _power(byte):
    """2^(byte - 127) in float32, from its bits (byte 0 gives a subnormal number)."""
    byte = byte.to(torch.int32)
    return torch.where(byte > 0, byte << 23, torch.full_like(byte, 1 << 22)).view(torch.float32)


def _quantized(x):
    """Float32 x -> (codes [..., 16 blocks], scales [..., blocks])."""
    b = _padded(x)
    top = b.abs().amax(-1)
    # (An exponent's field, less 2, is the scale's byte; subnormal numbers have field 0.)
    scales = torch.clamp((top.view(torch.int32) >> 23) - 2, min=0)
    v = b.abs() * _power(254 - scales)[..., None]
    codes = torch.zeros_like(v, dtype=torch.uint8)
    # A value halfway between two goes to the even code.
    for i, edge in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        codes += v > edge if i % 2 == 0 else v >= edge
    codes += (b < 0).to(torch.uint8) * 8
    fine = torch.isfinite(top)
    scales = torch.where(fine, scales, torch.full_like(scales, 255)).to(torch.uint8)
    codes = torch.where(fine[..., None], codes, torch.zeros_like(codes)).flatten(-2)
    return codes[..., 0::2] + codes[..., 1::2] * 16, scales


def _values(codes, scales, size):
    """The first `size` values that each row stands for."""
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    pair = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    factor = _power(scales)
    factor = torch.where(scales == 255, torch.full_like(factor, math.nan), factor)
    return (levels[pair.int()].unflatten(-1, (-1, 32)) * factor[..., None]).flatten(-2)[..., :size]


def _quant_plain(s):
    return {"y": _values(*_quantized(s["x"].float()), s["case"]["dim"]).to(s["x"].dtype)}


def _linear_plain(s):
    x, k = s["x"].float(), s["case"]["inputs"]
    if s["case"]["op"] == "linear4":
        x = _values(*_quantized(x), k)
    y = torch.matmul(x, _values(*s["weight"], k).t())
    if s["bias"] is not None:
        y = y + s["bias"]
    return {"y": y.to(s["x"].dtype)}


def _sequences(s):
    """(q [batch, tokens, heads, dim], each query's place in its sequence or -1, each sequence's and place's row of k and v)."""
    case, q = s["case"], s["q"]
    b, dev = case["batch"], q.device
    if case["step"]:
        n = torch.ones(b, dtype=torch.int64, device=dev)
        at = torch.arange(b, device=dev)[:, None]
    elif s["offsets"] is None:
        n = torch.full((b,), case["tokens"], device=dev)
        at = torch.arange(b, device=dev)[:, None] * case["tokens"] + torch.arange(case["tokens"], device=dev)
    else:
        n = (s["offsets"][1:] - s["offsets"][:-1]).long()
        at = s["offsets"][:-1, None].long() + torch.arange(s["max_len"], device=dev)
    i = torch.arange(at.shape[1], device=dev)
    place = torch.where(i < n[:, None], s["lengths"].long()[:, None] - n[:, None] + i, torch.full_like(at, -1))
    return place, torch.where(place >= 0, at, torch.zeros_like(at))


def _flat(t, lead):
    return t.flatten(0, lead - 1) if lead > 1 else t


def _attend_plain(s):
    case, page, dim = s["case"], s["case"]["page"], s["case"]["head_dim"]
    lead = s["q"].dim() - 2
    place, row = _sequences(s)
    live = place >= 0
    seq = torch.arange(case["batch"], device=place.device)[:, None].expand_as(place)
    p, r = place[live], row[live]
    block, off = s["tables"][seq[live], p // page].long(), p % page
    for j, name in enumerate("kv"):
        codes, scales = _quantized(_flat(s[name], lead)[r].float())
        s["cache"][2 * j][block, :, off] = codes
        s["cache"][2 * j + 1][block, :, off] = scales
    tables = torch.clamp(s["tables"], min=0).long()
    k, v = (_values(s["cache"][j][tables], s["cache"][j + 1][tables], dim).transpose(1, 2).flatten(2, 3) for j in (0, 2))
    q = _flat(s["q"], lead)[row].float()  # [batch, tokens, heads, dim]
    b, t, h, kv = q.shape[0], q.shape[1], q.shape[2], case["kv_heads"]
    q = q.transpose(1, 2).reshape(b, kv, h // kv * t, dim)
    there = torch.arange(k.shape[2], device=k.device) <= place[:, :, None]  # [batch, tokens, keys]
    # (What lies behind a sequence's last token counts for nothing, whatever it is.)
    ends = torch.arange(k.shape[2], device=k.device) < s["lengths"][:, None]
    k, v = (torch.where(ends[:, None, :, None], m, torch.zeros((), device=m.device)) for m in (k, v))
    w = torch.matmul(q * dim ** -0.5, k.transpose(-1, -2).contiguous()).view(b, h, t, -1)
    w.masked_fill_(~there[:, None], -math.inf)
    w -= torch.clamp(w.amax(-1, keepdim=True), min=-1e30)
    w.exp_()
    total = w.sum(-1, keepdim=True)
    y = torch.matmul(w.view(b, kv, h // kv * t, -1), v).view(b, h, t, dim)
    y = y / torch.where(total > 0, total, torch.ones_like(total))
    y = y.transpose(1, 2)
    y = y[:, 0] if case["step"] else y if s["offsets"] is None else y[live]
    return {"y": y.to(s["q"].dtype)}


def _grant(s, need):
    """Pages for requests that need `need` each, in turn, the lowest free ones first: (which get theirs, the
    free pages in order, each request's first)."""
    refs = s["refs"]
    free = refs == 0
    rank = torch.cumsum(free, 0) - 1
    order = torch.zeros(refs.numel() + 1, dtype=torch.int64, device=refs.device)
    order.scatter_(0, torch.where(free, rank, torch.full_like(rank, refs.numel())), torch.arange(refs.numel(), device=refs.device))
    ends = torch.cumsum(need, 0)
    return (ends <= free.sum()) | (need == 0), order, ends - need


def _copy(s, source, target):
    for pool in s["pools"]:
        pool[target] = pool[source]


def _resize_plain(s, rows, sizes):
    page, refs, tables, lengths = s["case"]["page"], s["refs"], s["tables"], s["lengths"]
    rows, sizes = rows.long(), sizes.long()
    old = lengths[rows].long()
    a, b = -(-old // page), -(-sizes // page)
    at = torch.arange(tables.shape[1], device=tables.device)
    mine = tables[rows]
    drop = (at >= b[:, None]) & (at < a[:, None])
    refs.index_add_(0, mine[drop].long(), torch.full_like(mine[drop], -1))
    mine[drop] = -1
    last = torch.clamp(mine.gather(1, torch.clamp(a - 1, min=0)[:, None])[:, 0], min=0).long()
    shared = (sizes > old) & (old % page > 0) & (refs[last] > 1)
    granted, order, first = _grant(s, torch.clamp(b - a, min=0) + shared)
    granted &= b <= tables.shape[1]
    shared &= granted
    fill = granted[:, None] & (at >= (a - shared.long())[:, None]) & (at < b[:, None])
    pages = order[torch.clamp(first[:, None] + at - (a - shared.long())[:, None], min=0, max=refs.numel())]
    mine[fill] = pages[fill].int()
    refs[pages[fill]] = 1
    refs.index_add_(0, last[shared], torch.full_like(last[shared], -1, dtype=torch.int32))
    _copy(s, last[shared], order[first[shared]])
    tables[rows] = mine
    lengths[rows] = torch.where(granted, sizes, old).int()
    return granted.int()


def _fork_plain(s, parents, children):
    page, refs, tables, lengths = s["case"]["page"], s["refs"], s["tables"], s["lengths"]
    parents, children = parents.long(), children.long()
    n = lengths[parents].long()
    part = (n % page > 0).long()
    granted, order, first = _grant(s, part)
    granted &= lengths[children] == 0
    at = torch.arange(tables.shape[1], device=tables.device)
    theirs = tables[parents]
    whole = granted[:, None] & (at < (n // page)[:, None])
    refs.index_add_(0, theirs[whole].long(), torch.ones_like(theirs[whole]))
    mine = torch.where(whole, theirs, torch.full_like(theirs, -1))
    copied = granted & (part > 0)
    last = (n // page)[copied]
    mine[copied, last] = order[first[copied]].int()
    refs[order[first[copied]]] = 1
    _copy(s, theirs[copied, last].long(), order[first[copied]])
    tables[children] = torch.where(granted[:, None], mine, tables[children])
    lengths[children] = torch.where(granted, n.int(), lengths[children])
    return granted.int()


def _compact_plain(s):
    refs, tables = s["refs"], s["tables"]
    used = refs > 0
    live = used.sum()
    at = torch.arange(refs.numel(), device=refs.device)
    hole, stray = ~used & (at < live), used & (at >= live)
    source, target = at[stray], at[hole]
    to = at.clone()
    to[source] = target
    _copy(s, source, target)
    refs[target] = refs[source]
    refs[source] = 0
    tables.copy_(torch.where(tables >= 0, to[torch.clamp(tables, min=0).long()].int(), tables))
    return live.int()


def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        resize, fork, compact = _resize_plain, _fork_plain, _compact_plain
        if op == "quant":
            return _quant_plain(s)
        if op in ("linear", "linear4"):
            return _linear_plain(s)
        if op == "attend":
            return _attend_plain(s)
    if own:
        from sparseflow_amd.Kernels.cached_attention import MX4Cache, cached_attention_forward, cached_attention_step, \
            mx4_cache_append
        from sparseflow_amd.Kernels.mx4 import mx4_dequantize, mx4_linear_forward, mx4_quantize
        from sparseflow_amd.Kernels.pages import pages_compact, pages_fork, pages_resize

        if op == "quant":
            codes, scales = mx4_quantize(s["x"])
            return {"y": mx4_dequantize(codes, scales, size=case["dim"], dtype=s["x"].dtype)}
        if op in ("linear", "linear4"):
            x = mx4_quantize(s["x"]) if op == "linear4" else s["x"]
            return {"y": mx4_linear_forward(x, s["weight"], bias=s["bias"], dtype=s["x"].dtype)}
        if op == "attend":
            cache = MX4Cache(*s["cache"])
            if case["step"]:
                mx4_cache_append(cache, s["k"][:, None], s["v"][:, None], s["tables"], s["lengths"])
                return {"y": cached_attention_step(s["q"], cache, s["tables"], s["lengths"])}
            mx4_cache_append(cache, s["k"], s["v"], s["tables"], s["lengths"], offsets=s["offsets"], max_len=s["max_len"])
            return {"y": cached_attention_forward(s["q"], cache, s["tables"], s["lengths"], offsets=s["offsets"],
                                                  max_len=s["max_len"])}

        def resize(s, rows, sizes):
            return pages_resize(s["refs"], s["tables"], s["lengths"], rows, sizes, case["page"], pools=s["pools"])

        def fork(s, parents, children):
            return pages_fork(s["refs"], s["tables"], s["lengths"], parents, children, case["page"], pools=s["pools"])

        def compact(s):
            return pages_compact(s["refs"], s["tables"], pools=s["pools"])[0]

    if op == "fork":
        before, after = s["rows"]
        granted = fork(s, before[s["picks"]], after)
        resize(s, before, s["none"])
        s["rows"] = [after, before]
        count = None
    else:
        ended = s["rows"][0]
        resize(s, ended, s["none"][0])
        count = compact(s)
        granted = resize(s, ended, s["sizes"][0])
        for name in ("rows", "sizes", "none"):
            s[name] = s[name][::-1]
    out = {"granted": granted, "refs": s["refs"], "tables": s["tables"], "lengths": s["lengths"], "pools": s["pools"]}
    if count is not None:
        out["live"] = count
    return out


def work(case):
    op = case["op"]
    if op == "quant":
        e, n, blocks = SIZE[case["dtype"]], case["rows"] * case["dim"], case["rows"] * _full(case["dim"], 32)
        return {"bytes": 2 * n * e + 2 * 17 * blocks, "flops": 4 * n}
    if op in ("linear", "linear4"):
        e, m, k, n = SIZE[case["dtype"]], case["rows"], case["inputs"], case["outputs"]
        quantised = 2 * m * 17 * _full(k, 32) if op == "linear4" else 0
        return {"bytes": e * m * (k + n) + 17 * n * _full(k, 32) + quantised + 4 * n * case["bias"], "flops": 2 * m * n * k}
    if op == "attend":
        new, old = _lengths(case)
        e, h, kv, dim = SIZE[case["dtype"]], case["heads"], case["kv_heads"], case["head_dim"]
        tokens, keys = sum(new), sum(new) + sum(old)
        pairs = sum(n * o + n * (n + 1) // 2 for n, o in zip(new, old))
        return {"bytes": tokens * e * dim * (2 * h + 2 * kv) + 2 * 17 * kv * _full(dim, 32) * (keys + tokens),
                "flops": 4 * dim * h * pairs}
    lens, page = _page_lengths(case), case["page"]
    bytes_of_page = 2 * 17 * page * case["kv_heads"] * _full(case["head_dim"], 32)
    held = [_full(n, page) for n in lens]
    if op == "fork":
        return {"bytes": 2 * bytes_of_page * case["rows"] + 24 * sum(held), "flops": 0}
    return {"bytes": 2 * bytes_of_page * min(sum(held[0::2]), sum(held[1::2])) + 24 * sum(held), "flops": 0}


# ---- the definitions, in 64 bits ----------------------------------------------


def _exact_scaled(v, e):
    """v 2^e in float64, the power from its bits."""
    return v * ((e.long() + 1023) << 52).view(torch.float64)


def _exact_values(x):
    """What the format makes of float64 x, in float64."""
    size = x.shape[-1]
    b = _padded(x)
    top = b.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(top)  # top = m 2^e, 1/2 <= m < 1
    e = torch.where(top > 0, e - 3, torch.full_like(e, -127)).clamp(min=-127)
    v = _exact_scaled(b, -e)
    # Steps of 1/2 below 2, of 1 below 4, of 2 from there; round() takes a half to the even side.
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(v.dtype)
    r = torch.clamp(torch.round(a / step) * step, max=6.0) * torch.sign(v)
    return _exact_scaled(r, e).flatten(-2)[..., :size]


def _exact_stored(codes, scales, size):
    magnitude = torch.tensor(LEVELS, dtype=torch.float64, device=codes.device)
    parts = []
    for half in (codes % 16, codes // 16):
        half = half.long()
        parts.append(magnitude[half % 8] * (1 - 2 * (half // 8)))
    v = torch.stack(parts, dim=-1).reshape(*scales.shape, 32)
    v = _exact_scaled(v, (scales.long() - 127)[..., None])
    v[scales == 255] = math.nan
    return v.reshape(*scales.shape[:-1], -1)[..., :size]


def exact(case, seed):
    op = case["op"]
    if op in ("fork", "compact"):
        return None  # whole numbers only
    s = prepare(case, seed)
    if op == "quant":
        return {"y": _exact_values(s["x"].double())}
    if op in ("linear", "linear4"):
        x = s["x"].double()
        if op == "linear4":
            x = _exact_values(x)
        y = x @ _exact_stored(*s["weight"], case["inputs"]).t().contiguous()
        return {"y": y if s["bias"] is None else y + s["bias"].double()}
    new, old = _lengths(case)
    if sum(n * (n + o) for n, o in zip(new, old)) * case["heads"] * case["head_dim"] > 2 ** 42:
        return None
    dim, page, group = case["head_dim"], case["page"], case["heads"] // case["kv_heads"]
    out, first = [], 0
    for i, (n, o) in enumerate(zip(new, old)):
        if case["step"] or s["offsets"] is None:
            q, k, v = (s[m][i].double().reshape(n, -1, dim) for m in "qkv")
        else:
            q, k, v = (s[m][first : first + n].double() for m in "qkv")
        first += n
        if n == 0:
            continue
        table = s["tables"][i, : _full(n + o, page)].long()
        past = [_exact_stored(s["cache"][j][table], s["cache"][j + 1][table], dim).transpose(0, 1).reshape(case["kv_heads"], -1, dim)[:, :o]
                for j in (0, 2)]
        k, v = (torch.cat([a, _exact_values(b).transpose(0, 1)], dim=1) for a, b in zip(past, (k, v)))
        ys = []
        for h in range(case["heads"]):
            for part in torch.arange(n, device=q.device).split(2048):
                w = q[part, h] @ k[h // group].t().contiguous() / math.sqrt(dim)
                hidden = torch.arange(n + o, device=q.device)[None] > (part + o)[:, None]
                ys.append(torch.softmax(w.masked_fill(hidden, -math.inf), dim=1) @ v[h // group])
        out.append(torch.cat(ys).reshape(case["heads"], n, dim).transpose(0, 1))
    if case["step"]:
        return {"y": torch.cat(out)}
    return {"y": torch.stack(out) if s["offsets"] is None else torch.cat(out)}
