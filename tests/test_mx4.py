"""The 4-bit operators without a GPU: the host forms against the 64-bit oracle, and the
refusals of the entry points and of the C ABI."""

import ctypes
import random

import pytest
import torch

from oracle import mx4 as ora
from sparseflow_amd import _lib
from sparseflow_amd.Kernels.cached_attention import MX4Cache, cached_attention_forward, cached_attention_step, mx4_cache, \
    mx4_cache_append
from sparseflow_amd.Kernels.mx4 import mx4_dequantize, mx4_linear_forward, mx4_quantize
from sparseflow_amd.Kernels.pages import pages_compact, pages_copy, pages_fork, pages_resize
from tests.mx4_checks import check_attention, check_linear, check_quantize, quantize_case
from tests.pages_checks import check_random_calls, start

CPU = torch.device("cpu")
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(5, 32), (7, 67), (4, 3, 100), (1, 1), (0, 40), (33,)])
def test_quantize(shape, dtype):
    check_quantize(quantize_case(CPU, shape, dtype))


def test_quantize_edges():
    x = torch.zeros(8, 40)
    x[0, 3] = float("inf")
    x[1, 39] = float("nan")
    x[2, 0] = 2.0 ** -149
    x[3, 0] = 3.4e38
    x[4, :3] = torch.tensor([2.0 ** -126, 2.0 ** -125, -2.0 ** -127])
    x[5] = -0.0
    x[6, 32:] = 1.0
    check_quantize(x)
    codes, scales = mx4_quantize(x)
    assert scales[0].tolist() == [255, 0] and scales[1].tolist() == [0, 255]
    spikes = (torch.rand(6, 70) < 0.2).float()
    assert torch.equal(mx4_dequantize(*mx4_quantize(spikes), size=70), spikes)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear(dtype):
    check_linear(CPU, 5, 67, 9, dtype, bias=True)
    check_linear(CPU, 1, 32, 1, dtype, four=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention(dtype):
    check_attention(CPU, [3, 0, 9, 1], [0, 5, 17, 8], 4, 2, 20, 8, dtype)
    check_attention(CPU, [4, 4], [0, 9], 3, 3, 33, 4, dtype, packed=False)
    check_attention(CPU, [1, 1, 1], [0, 30, 7], 6, 2, 16, 16, dtype, step=True)


@pytest.mark.parametrize("seed", range(6))
def test_pages_random_calls(seed):
    check_random_calls(CPU, seed)


def test_pages_shared_partial_page_is_copied_before_it_grows():
    s = start(CPU, pages=8, rows=4, width=4, page=4)
    r = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    assert pages_resize(s["refs"], s["tables"], s["lengths"], r(0), r(8), 4, s["pools"]).tolist() == [1]
    assert pages_fork(s["refs"], s["tables"], s["lengths"], r(0), r(1), 4, s["pools"]).tolist() == [1]
    assert s["refs"].tolist()[:3] == [2, 2, 0]
    assert pages_resize(s["refs"], s["tables"], s["lengths"], r(1), r(6), 4, s["pools"]).tolist() == [1]
    before = [p.clone() for p in s["pools"]]
    assert pages_resize(s["refs"], s["tables"], s["lengths"], r(1), r(7), 4, s["pools"]).tolist() == [1]
    assert s["tables"][1].tolist() == [0, 2, -1, -1] and s["refs"].tolist()[:3] == [2, 1, 1]
    for p, b in zip(s["pools"], before):
        assert torch.equal(p[2], b[1]) and torch.equal(p[1], b[1])


def test_refusals_of_quantize_and_linear():
    x = torch.randn(4, 70)
    w = mx4_quantize(torch.randn(6, 70))
    with pytest.raises(_lib.UnsupportedError):
        mx4_quantize(x.double())
    with pytest.raises(ValueError):
        mx4_quantize(torch.randn(()))
    with pytest.raises(ValueError):
        mx4_quantize(torch.zeros(3, 0))
    with pytest.raises(ValueError):
        mx4_quantize(x, out=(w[0], w[1]))
    for size in (64, 97, 0, -3):
        with pytest.raises(ValueError):
            mx4_dequantize(*w, size=size)
    with pytest.raises(ValueError):
        mx4_dequantize(w[0], w[1][:, :2])
    with pytest.raises(_lib.UnsupportedError):
        mx4_dequantize(*w, dtype=torch.float64)
    with pytest.raises(ValueError):
        mx4_dequantize(*w, size=70, out=torch.zeros(6, 71))
    ok = dict(x=x, weight=w)
    for kw in (dict(x=torch.randn(4, 97)), dict(weight=(w[0], w[1].int())), dict(weight=(w[0][:, :32], w[1])),
               dict(weight=w[0]), dict(bias=torch.randn(5)), dict(bias=torch.randn(6).half()), dict(x=(w[0], w[1], w[1])),
               dict(x=mx4_quantize(torch.randn(4, 32))), dict(out=torch.zeros(4, 7)), dict(out=torch.zeros(6, 4).t()),
               dict(out=torch.zeros(1, 6).expand(4, 6)), dict(out=torch.zeros(4, 6), dtype=torch.half),
               dict(weight=(w[0][None], w[1][None])), dict(x=torch.randn(())), dict(x=())):
        with pytest.raises(ValueError):
            mx4_linear_forward(**{**ok, **kw})
    for kw in (dict(x=x.double()), dict(dtype=torch.float64)):
        with pytest.raises(_lib.UnsupportedError):
            mx4_linear_forward(**{**ok, **kw})
    both = torch.zeros(4, 76)
    with pytest.raises(ValueError):
        mx4_linear_forward(both[:, :70], w, out=both[:, 68:74])
    assert torch.equal(mx4_linear_forward(both[:, :70], w, out=both[:, 70:]), torch.zeros(4, 6))


def test_refusals_of_attention():
    cache = mx4_cache(6, 2, 8, 20)
    tables, lengths = torch.full((3, 2), -1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    k, q = torch.randn(3, 2, 2, 20), torch.randn(3, 2, 4, 20)
    mx4_cache_append(cache, k, k, tables, lengths)
    assert not cached_attention_forward(q, cache, tables, lengths).any()
    i = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    bad_k = (dict(k=k[0]), dict(v=k[:, :1]), dict(v=k.half()), dict(k=k[:, :, :1], v=k[:, :, :1]), dict(k=k[..., :10], v=k[..., :10], cache=mx4_cache(6, 2, 8, 40)),
             dict(tables=tables.long()), dict(tables=tables[:2]), dict(lengths=lengths[:2]), dict(slots=i(0, 1)),
             dict(slots=torch.zeros(3)), dict(cache=MX4Cache(cache.k, cache.v, cache.v, cache.v_scales)), dict(tables=tables.t()),
             dict(offsets=i(0, 1)), dict(cache=cache[:3]))
    for kw in bad_k:
        with pytest.raises(ValueError):
            mx4_cache_append(**{**dict(cache=cache, k=k, v=k, tables=tables, lengths=lengths), **kw})
    for kw in (dict(q=q[0]), dict(q=q[:, :, :3]), dict(q=q[..., :0]), dict(out=torch.zeros(3, 2, 4, 21)),
               dict(out=torch.zeros(3, 2, 4, 20).half()), dict(out=torch.zeros(3, 2, 20, 4).transpose(2, 3)),
               dict(out=torch.zeros(1, 2, 4, 20).expand(3, -1, -1, -1)), dict(q=q.flatten(0, 1), offsets=i())):
        with pytest.raises(ValueError):
            cached_attention_forward(**{**dict(q=q, cache=cache, tables=tables, lengths=lengths), **kw})
    with pytest.raises(_lib.UnsupportedError):
        cached_attention_forward(q.double(), cache, tables, lengths)
    with pytest.raises(_lib.UnsupportedError):
        cached_attention_forward(torch.randn(3, 2, 4, 257), mx4_cache(6, 2, 8, 257), tables, lengths)
    for page in (6, 8192):
        with pytest.raises(_lib.UnsupportedError):
            cached_attention_forward(q, mx4_cache(2, 2, page, 20), tables, lengths)
    with pytest.raises(ValueError):
        cached_attention_step(q, cache, tables, lengths)


def test_refusals_of_pages():
    s = start(CPU, pages=8, rows=4, width=4, page=4)
    i = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    ok = dict(refs=s["refs"], tables=s["tables"], lengths=s["lengths"], rows=i(0), sizes=i(3), page_size=4, pools=s["pools"])
    for kw in (dict(refs=s["refs"].long()), dict(tables=s["tables"][0]), dict(lengths=i(0)), dict(rows=i(0, 1)), dict(page_size=0),
               dict(sizes=torch.tensor([3])), dict(pools=[torch.zeros(7, 3)]), dict(pools=[torch.zeros(3, 8).t()]),
               dict(rows=s["lengths"][:1]), dict(pools=[s["pools"][0], s["pools"][0]])):
        with pytest.raises(ValueError):
            pages_resize(**{**ok, **kw})
    with pytest.raises(_lib.UnsupportedError):
        pages_resize(**{**ok, "pools": [torch.zeros(8, 1) for _ in range(17)]})
    with pytest.raises(ValueError):
        pages_fork(s["refs"], s["tables"], s["lengths"], i(0), i(1, 2), 4)
    with pytest.raises(ValueError):
        pages_compact(s["refs"][None], s["tables"])
    for args in (([], i(0), i(1)), (s["pools"], i(0), i(1, 2)), (s["pools"], torch.tensor([0]), i(1))):
        with pytest.raises(ValueError):
            pages_copy(*args)


def test_c_abi_refusals():
    L = _lib.lib()
    one = ctypes.c_void_p(16)
    st = (ctypes.c_int64 * 2)(0, 32)
    at = ctypes.addressof
    assert L.sf_mx4_quantize(one, 7, 1, 1, at(st), 32, one, one, None) == _lib.SF_ERR_INVALID
    assert L.sf_mx4_quantize(one, 0, 1, -1, at(st), 32, one, one, None) == _lib.SF_ERR_INVALID
    assert L.sf_mx4_quantize(one, 0, 1, 1, at(st), 32, ctypes.c_void_p(8), one, None) == _lib.SF_ERR_INVALID
    assert L.sf_mx4_quantize(one, 0, 0, 1, at(st), 32, one, one, None) == _lib.SF_OK
    assert L.sf_mx4_dequantize(one, one, 1, 0, one, 0, None) == _lib.SF_ERR_INVALID
    assert L.sf_mx4_dequantize(one, None, 1, 4, one, 0, None) == _lib.SF_ERR_INVALID
    d = _lib.Mx4LinearDesc(1, 4, 4, 4, 4, 0, 0)
    assert L.sf_mx4_linear(None, one, None, one, one, None, one, None) == _lib.SF_ERR_INVALID
    assert L.sf_mx4_linear(at(d), one, one, one, one, None, one, None) == _lib.SF_ERR_INVALID  # scales of floats
    d.x_dtype = 9
    assert L.sf_mx4_linear(at(d), one, None, one, one, None, one, None) == _lib.SF_ERR_INVALID
    zero = (0, 0, 0)
    c = _lib.Mx4CacheDesc(1, 1, 1, 1, 1, 1, zero, zero, zero, zero, 4, 2, 20, 8, 0, 1.0)
    t = _lib.Mx4CacheTensors(16, 16, 16, 16, 16, 16)
    call = lambda: L.sf_mx4_attention(at(c), at(t), one, None, None, one, None, 0, None)  # noqa: E731
    for name, value, code in (("heads", 3, 1), ("dtype", 5, 1), ("head_dim", 257, 2), ("page_size", 6, 2), ("rows", -1, 1),
                              ("page_size", 8192, 2), ("width", 1 << 31, 2)):
        was = getattr(c, name)
        setattr(c, name, value)
        assert call() == code, name
        setattr(c, name, was)
    t.k = 8
    assert call() == _lib.SF_ERR_INVALID
    t.k = 16
    c.width = 4096
    assert L.sf_mx4_attention_workspace_size(at(c)) > 0 and call() == _lib.SF_ERR_WORKSPACE
    p = _lib.PagesDesc(4, 2, 2, 1, 4, 0)
    assert L.sf_pages_resize(at(p), one, one, one, one, one, one, None, 0, None) == _lib.SF_ERR_WORKSPACE
    p.pools = 17
    assert L.sf_pages_resize(at(p), one, one, one, one, one, one, one, 1 << 20, None) == _lib.SF_ERR_UNSUPPORTED
    p.pools, p.page_size = 0, 0
    assert L.sf_pages_copy(at(p), one, one, None) == _lib.SF_ERR_INVALID
