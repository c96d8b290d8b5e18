"""Random calls of the page operators against the oracle's lists."""

import random

import torch

from oracle import mx4 as ora
from sparseflow_amd.Kernels.pages import pages_compact, pages_copy, pages_fork, pages_resize


def start(dev, pages, rows, width, page, seed=0):
    g = torch.Generator().manual_seed(seed)
    pools = [torch.randint(0, 256, (pages, 2, page, n), generator=g, dtype=torch.uint8).to(dev) for n in (16, 1, 3)]
    pools.append(torch.randn(pages, 5, generator=g).to(dev))
    return dict(refs=torch.zeros(pages, dtype=torch.int32, device=dev), lengths=torch.zeros(rows, dtype=torch.int32, device=dev),
                tables=torch.full((rows, width), -1, dtype=torch.int32, device=dev), pools=pools)


def same(s, model, names):
    assert s["refs"].tolist() == model.refs and s["lengths"].tolist() == model.lengths
    assert s["tables"].tolist() == model.tables()
    for i, pool in enumerate(s["pools"]):
        for p, (was, r) in enumerate(zip(model.contents, model.refs)):
            if r > 0:  # (what a free page holds is nobody's)
                assert torch.equal(pool[p].cpu(), names[was][i]), (i, p)


def check_random_calls(dev, seed, calls=25, pages=23, rows=9, width=6):
    rng = random.Random(seed)
    page = rng.choice([1, 3, 4, 8])
    s = start(dev, pages, rows, width, page, seed)
    names = {p: [t[p].cpu().clone() for t in s["pools"]] for p in range(pages)}
    model = ora.Pages(s["refs"], s["tables"], s["lengths"], page, range(pages))
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    refused = 0
    for _ in range(calls):
        op = rng.choice(["resize", "resize", "resize", "fork", "fork", "compact", "copy"])
        if op == "resize":
            n = rng.randint(0, 6)
            a, b = [rng.randint(-1, rows) for _ in range(n)], [rng.randint(-2, width * page + 2) if rng.random() < 0.7 else 0 for _ in range(n)]
            got = pages_resize(s["refs"], s["tables"], s["lengths"], ints(a), ints(b), page, s["pools"])
            assert got.tolist() == model.resize(a, b)
            refused += n - int(got.sum())
        elif op == "fork":
            n = rng.randint(0, 6)
            a, b = [rng.randint(-1, rows) for _ in range(n)], [rng.randint(-1, rows) for _ in range(n)]
            got = pages_fork(s["refs"], s["tables"], s["lengths"], ints(a), ints(b), page, s["pools"])
            assert got.tolist() == model.fork(a, b)
        elif op == "compact":
            assert pages_compact(s["refs"], s["tables"], s["pools"]).tolist() == [model.compact()]
        else:
            free = [p for p in range(pages) if model.refs[p] == 0]
            live = [p for p in range(pages) if model.refs[p] > 0]
            pairs = list(zip(live, free))[:3]
            pages_copy(s["pools"], ints([p for p, _ in pairs] + [-1, 0]), ints([p for _, p in pairs] + [0, pages]))
            for a, b in pairs:
                model.contents[b] = model.contents[a]
                for pool in s["pools"]:
                    assert torch.equal(pool[a], pool[b])
        same(s, model, names)
    return refused
