"""Page calls on the GPU whose requests, times the workgroups that copy a page, are more than one launch holds."""

import pytest
import torch

from sparseflow_amd.Kernels.pages import pages_copy, pages_fork, pages_resize
from tests.gpu_helpers import DEV, announce

pytestmark = pytest.mark.gpu


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _pool(pages):
    """Pages of a megabyte: 64 workgroups to a copy."""
    return torch.randint(0, 256, (pages, 1 << 20), dtype=torch.uint8, generator=torch.Generator().manual_seed(pages)).to(DEV)


def test_copies():
    announce("pages_copy of 300,000 pairs")
    pool = _pool(5)
    was = pool.clone()
    sources, targets = torch.full((300000,), -1, dtype=torch.int32, device=DEV), torch.full((300000,), 9, dtype=torch.int32, device=DEV)
    sources[5], targets[5] = 1, 3
    sources[150000], targets[150000] = 4, 0
    sources[299999], targets[299999] = 1, 2
    pages_copy([pool], sources, targets)
    assert torch.equal(pool, was[[4, 1, 1, 1, 4]])


def test_resizes():
    """The last request is the one that has to have a page copied."""
    announce("pages_resize of 70,000 rows")
    rows, pages = 70000, 8
    pool = _pool(pages)
    was = pool.clone()
    refs, lengths = torch.zeros(pages, dtype=torch.int32, device=DEV), torch.zeros(rows, dtype=torch.int32, device=DEV)
    tables = torch.full((rows, 2), -1, dtype=torch.int32, device=DEV)
    refs[6], tables[0, 0], tables[1, 0], lengths[:2] = 2, 6, 6, 3
    order = torch.cat([torch.arange(2, rows, device=DEV), torch.tensor([0, 1], device=DEV)]).int()
    sizes = torch.zeros(rows, dtype=torch.int32, device=DEV)
    sizes[7], sizes[40000], sizes[-2], sizes[-1] = 5, 4, 3, 4
    granted = pages_resize(refs, tables, lengths, order, sizes, 4, [pool])
    assert bool((granted == 1).all())
    assert refs.tolist() == [1, 1, 1, 1, 0, 0, 1, 0]
    assert tables[9].tolist() == [0, 1] and tables[40002].tolist() == [2, -1] and tables[1].tolist() == [3, -1]
    assert tables[0].tolist() == [6, -1] and lengths[[0, 1, 9, 40002]].tolist() == [3, 4, 5, 4] and int(lengths.sum()) == 16
    assert torch.equal(pool, was[[0, 1, 2, 6, 4, 5, 6, 7]])


def test_forks():
    announce("pages_fork of 70,000 requests")
    rows, pages = 70000, 8
    pool = _pool(pages)
    was = pool.clone()
    refs, lengths = torch.zeros(pages, dtype=torch.int32, device=DEV), torch.zeros(rows, dtype=torch.int32, device=DEV)
    tables = torch.full((rows, 2), -1, dtype=torch.int32, device=DEV)
    refs[6], refs[2], lengths[0] = 1, 1, 7
    tables[0] = _ints(6, 2)
    parents, children = torch.ones(rows, dtype=torch.int32, device=DEV), torch.arange(rows, dtype=torch.int32, device=DEV)
    parents[3], parents[-1] = 0, 0
    granted = pages_fork(refs, tables, lengths, parents, children, 4, [pool])
    assert granted.tolist() == [0] + [1] * (rows - 1)  # (row 0 is not empty)
    assert refs.tolist() == [1, 1, 1, 0, 0, 0, 3, 0]
    assert tables[3].tolist() == [6, 0] and tables[-1].tolist() == [6, 1] and int(lengths.sum()) == 21
    assert torch.equal(pool, was[[2, 2, 2, 3, 4, 5, 6, 7]])
