"""The 4-bit operators on the GPU against the 64-bit oracle and the host forms."""

import pytest
import torch

from oracle import mx4 as ora
from sparseflow_amd.Kernels.cached_attention import MX4Cache, cached_attention_forward, cached_attention_step, mx4_cache, \
    mx4_cache_append
from sparseflow_amd.Kernels.mx4 import mx4_dequantize, mx4_linear_forward, mx4_quantize
from sparseflow_amd.Kernels.pages import pages_compact, pages_copy, pages_fork, pages_resize
from tests.gpu_helpers import DEV, announce, native_loaded
from tests.mx4_checks import attention_bound, attention_case, check_attention, check_linear, check_quantize, half_step, quantize_case, within
from tests.pages_checks import check_random_calls, start

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


# ---- quantisation ---------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(5, 32), (7, 67), (4, 3, 100), (1, 1), (0, 40), (33,), (300, 129), (3, 4097)])
def test_quantize(shape, dtype):
    announce(f"quantize {shape} {dtype}")
    check_quantize(quantize_case(DEV, shape, dtype))
    assert native_loaded()


def test_quantize_every_exponent_and_the_edges():
    x = torch.zeros(260, 40)
    x[:255, 0] = torch.ldexp(torch.ones(255), torch.arange(-127, 128).clamp(-149, 127).int()) * 1.25
    x[:255, 1:33] = x[:255, :1] * torch.rand(255, 32)
    x[255, 3] = float("-inf")
    x[256, 39] = float("nan")
    x[257, 0] = 2.0 ** -149
    x[258, 0] = 3.4e38
    x[259] = -0.0
    check_quantize(x.to(DEV))


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_views(dtype):
    """Rows anywhere: a slice of wider rows, transposed axes, an odd first element, expanded rows."""
    base = quantize_case(DEV, (6, 5, 4, 133), dtype)
    flat = base.flatten()
    for x in (base[1:, :, :, 3:70], base.transpose(0, 1), base.permute(2, 0, 1, 3), flat[1:1 + 7 * 65].view(7, 65),
              base[:1, :1].expand(3, 5, 4, 133), base[..., 0], base[..., ::2]):
        check_quantize(x)
    out = (torch.zeros(6, 5, 4, 80, dtype=torch.uint8, device=DEV), torch.zeros(6, 5, 4, 5, dtype=torch.uint8, device=DEV))
    got = mx4_quantize(base, out=out)
    assert got[0] is out[0] and torch.equal(out[0], mx4_quantize(base)[0]) and torch.equal(out[1], mx4_quantize(base)[1])


# ---- Linear -----------------------------------------------------------------------

SHAPES = [(1, 32, 1), (1, 4096, 64), (3, 67, 33), (16, 1000, 130), (17, 128, 16), (37, 1000, 1037), (64, 256, 256), (65, 320, 129),
          (128, 160, 500), (257, 96, 300), (300, 1056, 257), (513, 512, 512)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("four", [False, True], ids=["floats", "4-bit"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_linear(shape, dtype, four):
    announce(f"linear {shape} {dtype} {four}")
    m, k, n = shape
    check_linear(DEV, m, k, n, dtype, bias=m % 2 == 1, four=four)


@pytest.mark.parametrize("m", [5, 200])
def test_linear_views_and_types(m):
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(m, 3, 171, generator=g).to(DEV)
    for dtype in TYPES:
        x = wide.to(dtype)
        check_linear(DEV, m, 101, 70, dtype, x=x[:, 1, 7:108], bias=True)
        check_linear(DEV, m, 101, 70, dtype, x=x[:, 1, 7:108], out_dtype=torch.float32)
    w = mx4_quantize(torch.randn(40, 101, generator=g).to(DEV))
    x = wide[:, :, 7:108]
    ref = mx4_linear_forward(x.contiguous(), w)
    assert torch.equal(mx4_linear_forward(x, w), ref) and ref.shape == (m, 3, 40)
    out = torch.full((m, 3, 50), 7.0, device=DEV)
    mx4_linear_forward(x.contiguous(), w, out=out[..., 5:45])
    assert torch.equal(out[..., 5:45], ref) and bool((out[..., :5] == 7).all()) and bool((out[..., 45:] == 7).all())
    assert mx4_linear_forward(x[:0].contiguous(), w).shape == (0, 3, 40)


@pytest.mark.parametrize("m", [3, 150])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_numbers_that_are_none(m, dtype):
    """Infinities and NaN stay in their row, weights that are none in their column."""
    g = torch.Generator().manual_seed(5)
    w = torch.randn(150, 70, generator=g)
    w = (w.sign() * (w.abs() + 0.3)).to(DEV)  # no weight is 0
    x = torch.randn(m, 70, generator=g).to(dtype).to(DEV)
    q = mx4_quantize(w)
    clean = mx4_linear_forward(x, q)
    x[0, 3], x[1, 69] = float("inf"), float("nan")
    y = mx4_linear_forward(x, q)
    sign = ora.values(*q, 70)[:, 3]
    assert torch.equal(y[0].cpu().double(), torch.where(sign == 0, torch.nan, sign * float("inf")).double()) or bool((sign == 0).any())
    assert torch.isnan(y[1]).all() and torch.equal(y[2:], clean[2:])
    x4 = mx4_quantize(x)
    y = mx4_linear_forward(x4, q)
    assert torch.isnan(y[:2]).all() and torch.isfinite(y[2:]).all()
    w[5, 40] = float("nan")
    y = mx4_linear_forward(x[2:], mx4_quantize(w))
    assert torch.isnan(y[:, 5]).all() and torch.equal(y[:, :5], clean[2:, :5]) and torch.equal(y[:, 6:], clean[2:, 6:])


@pytest.mark.parametrize("m", [2, 140])
def test_linear_far_scales(m):
    """Weights and activations at the ends of the range: the scales of a block are any power of two."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(m, 96, generator=g)
    w = torch.randn(33, 96, generator=g)
    for a, b in ((100, -110), (-100, 100), (60, 60), (-60, -50)):
        for dtype in (torch.float32, torch.bfloat16):
            check = (x * 2.0 ** a).to(dtype).to(DEV)
            q = mx4_quantize((w * 2.0 ** b).to(DEV))
            y = mx4_linear_forward(check, q, dtype=torch.float32)
            ref, mag = ora.linear(check, ora.values(*q, 96))
            within(y, ref, (3 * 96 + 4) * 2.0 ** -23 * mag + 2.0 ** -24 * ref.abs(), f"{a} {b} {dtype}")


def test_spikes_are_exact():
    x = (torch.rand(40, 96, generator=torch.Generator().manual_seed(1)) < 0.1).float().to(DEV)
    w = mx4_quantize(torch.randn(64, 96, generator=torch.Generator().manual_seed(2)).to(DEV))
    four = mx4_linear_forward(mx4_quantize(x), w)
    ref, mag = ora.linear(x, ora.values(*w, 96))
    within(four, ref, 100 * 2.0 ** -23 * mag, "spikes")


# ---- attention ----------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 20, 33, 64, 80, 128, 131, 180, 200, 256])
def test_attention_head_dims(dim, dtype):
    announce(f"attention dim {dim} {dtype}")
    check_attention(DEV, [3, 0, 9, 1, 40], [0, 5, 57, 88, 0], 4, 2, dim, 8, dtype)
    check_attention(DEV, [1, 1, 1, 1], [0, 130, 7, 31], 6, 2, dim, 16, dtype, step=True)


@pytest.mark.parametrize("page", [1, 2, 16, 128, 4096])
@pytest.mark.parametrize("heads, kv", [(1, 1), (3, 3), (7, 1), (16, 1), (40, 2)])
def test_attention_pages_and_groups(heads, kv, page):
    check_attention(DEV, [5, 31, 1], [70, 0, 33], heads, kv, 64, page, torch.bfloat16)
    check_attention(DEV, [1, 1], [300, 2], heads, kv, 32, page, torch.float16, step=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_prompts(dtype):
    check_attention(DEV, [130, 130], [0, 0], 4, 2, 64, 16, dtype, packed=False)
    check_attention(DEV, [257, 5, 0, 128], [100, 0, 9, 129], 2, 1, 128, 64, dtype)


def test_attention_long_context_in_parts():
    """A sequence whose tokens are cut into parts (small against the many that are launched)."""
    check_attention(DEV, [1], [5000], 4, 2, 64, 16, torch.float16, step=True)
    check_attention(DEV, [3], [3333], 4, 1, 128, 64, torch.float32)


@pytest.mark.parametrize("n", [1, 37, 200])
def test_attention_odd_rows(n):
    """Slots outside the tables, empty sequences, pages that are none, lengths past the table: zeros or fewer tokens, and
    rows of no sequence left as they were."""
    call, held, q = attention_case(DEV, [n, n, n], [50, 20, 9], 4, 2, 64, 16, torch.float32, False)
    base = cached_attention_forward(**call)
    slots = torch.tensor([2, -1, 5], dtype=torch.int32, device=DEV)
    y = cached_attention_forward(**{**call, "q": call["q"][[2, 1, 0]].contiguous()}, slots=slots)
    assert torch.equal(y[0], base[2]) and not y[1:].any()
    lengths = call["lengths"].clone()
    lengths[1] = 0
    y = cached_attention_forward(**{**call, "lengths": lengths})
    assert torch.equal(y[0], base[0]) and not y[1].any()
    lengths[1] = -5
    assert not cached_attention_forward(**{**call, "lengths": lengths})[1].any()
    # No page where the first 16 tokens are: they are seen by nobody.
    tables = call["tables"].clone()
    tables[0, 0], tables[1, 0] = -1, 1 << 20
    y = cached_attention_forward(**{**call, "tables": tables})
    assert torch.isfinite(y).all() and not torch.equal(y[0], base[0]) and torch.equal(y[2], base[2])
    host = MX4Cache(*(t.cpu() for t in call["cache"]))
    ref = cached_attention_forward(call["q"].cpu(), host, tables.cpu(), call["lengths"].cpu())
    within(y, ref.double(), torch.full(ref.shape, 1e-4, dtype=torch.float64), "no page")  # float32 both, |v| < 8, 250 tokens
    # Packed rows of no sequence.
    qp = call["q"].flatten(0, 1)
    out = torch.full_like(qp, 7.0)
    off = torch.tensor([n, 2 * n, 2 * n], dtype=torch.int32, device=DEV)
    cached_attention_forward(qp, call["cache"], call["tables"][:2], call["lengths"][[1, 0]].contiguous(), offsets=off, out=out)
    assert bool((out[:n] == 7).all()) and bool((out[2 * n:] == 7).all())


@pytest.mark.parametrize("n", [1, 40, 150])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_numbers_that_are_none_stay_behind_the_mask(n, dtype):
    """A NaN key or value reaches the queries that see its token, and no other."""
    call, held, q = attention_case(DEV, [n], [45], 2, 1, 64, 16, dtype, False)
    base = cached_attention_forward(**call)
    t = 45 + n // 2
    page, row = int(call["tables"][0, t // 16]), t % 16
    for name in ("v_scales", "k_scales"):
        cache = MX4Cache(*(x.clone() for x in call["cache"]))
        getattr(cache, name)[page, 0, row, 1] = 255
        y = cached_attention_forward(**{**call, "cache": cache})
        assert torch.equal(y[0, :n // 2], base[0, :n // 2]) or float((y[0, :n // 2].float() - base[0, :n // 2].float()).abs().max()) < 2e-2
        hit = y[0, n // 2:]
        if name == "v_scales":
            assert torch.isnan(hit[..., 32:]).all() and torch.isfinite(hit[..., :32]).all()
        else:
            assert torch.isnan(hit).all()
    q = call["q"].clone()
    q[0, n // 2, 1, 3] = float("nan")
    y = cached_attention_forward(**{**call, "q": q})
    assert torch.isnan(y[0, n // 2, 1]).all()
    keep = torch.ones(n, 2, dtype=torch.bool, device=DEV)
    keep[n // 2, 1] = False
    assert torch.equal(y[0][keep], base[0][keep])


def test_append_views_places_and_slots():
    """Slices of a projection, a token without a place, rows that are no sequence's; what else the cache holds stays."""
    g = torch.Generator().manual_seed(4)
    for dtype in TYPES:
        qkv = torch.randn(2, 5, 8, 40, generator=g).to(dtype)
        k, v = qkv[:, :, 4:6, 3:36], qkv[:, :, 6:8, 3:36]
        tables = torch.tensor([[3, -1, 0], [9, 2, 7], [1, 5, 4]], dtype=torch.int32)
        lengths = torch.tensor([3, 12, 10], dtype=torch.int32)
        slots = torch.tensor([0, 2], dtype=torch.int32)
        caches = [MX4Cache(*(t.fill_(17) for t in mx4_cache(10, 2, 4, 33, device=d))) for d in ("cpu", DEV)]
        mx4_cache_append(caches[0], k, v, tables, lengths, slots=slots)
        dk, dv = qkv.to(DEV)[:, :, 4:6, 3:36], qkv.to(DEV)[:, :, 6:8, 3:36]
        mx4_cache_append(caches[1], dk, dv, tables.to(DEV), lengths.to(DEV), slots=slots.to(DEV))
        for a, b in zip(*caches):
            assert torch.equal(a, b.cpu())
        for out in (torch.tensor([5, 1], dtype=torch.int32), torch.tensor([-1, 3], dtype=torch.int32)):
            before = [t.clone() for t in caches[1]]
            if int(out[1]) == 1:
                mx4_cache_append(caches[0], k, v, tables, lengths, slots=out)
            mx4_cache_append(caches[1], dk, dv, tables.to(DEV), lengths.to(DEV), slots=out.to(DEV))
            if int(out[1]) == 3:
                for a, b in zip(caches[1], before):
                    assert torch.equal(a, b)
            else:
                for a, b in zip(*caches):
                    assert torch.equal(a, b.cpu())


def test_attention_places_past_32_bits():
    """A pool whose codes pass 4 GB: rows on both sides of the border."""
    pages, page, kv, dim = 2200, 4096, 4, 256  # 4.6 GB of codes each for keys and values
    cache = MX4Cache(*(torch.empty(pages, kv, page, n, dtype=torch.uint8, device=DEV) for n in (128, 8, 128, 8)))
    g = torch.Generator().manual_seed(8)
    k, v = (torch.randn(1, 40, kv, dim, generator=g).to(DEV) for _ in "kv")
    q = torch.randn(1, 3, 8, dim, generator=g).to(DEV)
    ys = []
    for places in ([0], [pages - 1], [2047], [2048]):
        tables = torch.tensor([places], dtype=torch.int32, device=DEV)
        lengths = torch.tensor([40], dtype=torch.int32, device=DEV)
        mx4_cache_append(cache, k, v, tables, lengths)
        ys.append(cached_attention_forward(q, cache, tables, lengths))
    for y in ys[1:]:
        assert torch.equal(y, ys[0])
    pages_copy(cache, torch.tensor([pages - 1], dtype=torch.int32, device=DEV), torch.tensor([7], dtype=torch.int32, device=DEV))
    assert torch.equal(cached_attention_forward(q, cache, torch.tensor([[7]], dtype=torch.int32, device=DEV), lengths), ys[0])


def test_out_may_be_q():
    call, _, _ = attention_case(DEV, [33, 33], [7, 40], 4, 2, 64, 16, torch.bfloat16, False)
    base = cached_attention_forward(**call)
    cached_attention_forward(**call, out=call["q"])
    assert torch.equal(call["q"], base)
    call, _, q = attention_case(DEV, [1, 1], [7, 900], 4, 2, 64, 16, torch.bfloat16, False)
    base = cached_attention_step(q, call["cache"], call["tables"], call["lengths"])
    cached_attention_step(q, call["cache"], call["tables"], call["lengths"], out=q)
    assert torch.equal(q, base)


# ---- pages --------------------------------------------------------------------------


@pytest.mark.parametrize("seed", range(8))
def test_pages_random_calls(seed):
    check_random_calls(DEV, seed)


def test_pages_many_requests():
    check_random_calls(DEV, 100, calls=12, pages=5000, rows=40, width=300)
    s = start(DEV, pages=9000, rows=3000, width=5, page=2)
    rows = torch.arange(3000, dtype=torch.int32, device=DEV)
    sizes = (rows % 7).int()
    host = start(torch.device("cpu"), pages=9000, rows=3000, width=5, page=2)
    for size in (sizes, (rows % 4).int(), torch.full_like(rows, 7), torch.full_like(rows, 10), torch.zeros_like(rows)):
        a = pages_resize(s["refs"], s["tables"], s["lengths"], rows, size, 2, s["pools"])
        b = pages_resize(host["refs"], host["tables"], host["lengths"], rows.cpu(), size.cpu(), 2, host["pools"])
        assert torch.equal(a.cpu(), b)
        for name in ("refs", "tables", "lengths"):
            assert torch.equal(s[name].cpu(), host[name]), name


# ---- together, as they are used -------------------------------------------------------


def _serving(dev, calls=None):
    """Prompts into fresh pages, a fork, steps of one token, an end, a compaction: every output."""
    g = torch.Generator().manual_seed(11)
    page, kv, heads, dim = 8, 2, 4, 64
    cache = mx4_cache(40, kv, page, dim, device=dev)
    s = start(dev, pages=40, rows=6, width=9, page=page)
    refs, tables, lengths = s["refs"], s["tables"], s["lengths"]
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    r = lambda *n: torch.randn(*n, generator=g).to(torch.bfloat16).to(dev)  # noqa: E731
    w = mx4_quantize(torch.randn(heads * dim, heads * dim, generator=g).to(dev) / 16)
    ys = []
    pages_resize(refs, tables, lengths, i(0, 3), i(19, 9), page, cache)
    off = i(0, 19, 28)
    mx4_cache_append(cache, r(28, kv, dim), r(28, kv, dim), tables, lengths, slots=i(0, 3), offsets=off)
    y = cached_attention_forward(r(28, heads, dim), cache, tables, lengths, slots=i(0, 3), offsets=off, max_len=19)
    ys.append(mx4_linear_forward(y.flatten(1), w))
    pages_fork(refs, tables, lengths, i(0, 0), i(1, 2), page, cache)
    live = i(0, 1, 2, 3)
    for t in range(6):
        grown = lengths[:4] + 1
        ys.append(pages_resize(refs, tables, lengths, live, grown.contiguous(), page, cache))
        mx4_cache_append(cache, r(4, 1, kv, dim), r(4, 1, kv, dim), tables, lengths, slots=live)
        y = cached_attention_step(r(4, heads, dim), cache, tables, lengths, slots=live)
        ys.append(mx4_linear_forward(mx4_quantize(y.flatten(1)), w, dtype=y.dtype))
    pages_resize(refs, tables, lengths, i(0), i(0), page, cache)
    ys.append(pages_compact(refs, tables, cache))
    ys.append(cached_attention_step(r(3, heads, dim), cache, tables, lengths, slots=i(1, 2, 3)))
    return ys + [refs, tables, lengths]


def test_serving_together():
    for a, b in zip(_serving(DEV), _serving(torch.device("cpu"))):
        if a.dtype == torch.int32:
            assert torch.equal(a.cpu(), b)
        else:
            # Both round a result and what it is made of (attention's output, in 4 bits for the steps) from sums of their
            # own: a few in a thousand fall to the other side of a rounding.
            d = (a.cpu().float() - b.float()).norm() / b.float().norm()
            assert float(d) < 2e-2


def test_captured_steps_replay():
    """A serving step in a graph: replays with eager work between them, each against the eager result."""
    g = torch.Generator().manual_seed(12)
    page, kv, heads, dim, n = 8, 2, 4, 64, 3
    make = lambda: (mx4_cache(40, kv, page, dim, device=DEV), start(DEV, pages=40, rows=n, width=9, page=page))  # noqa: E731
    r = lambda *v: torch.randn(*v, generator=g).to(torch.float16).to(DEV)  # noqa: E731
    w = mx4_quantize(torch.randn(48, heads * dim, generator=g).to(DEV))
    rows = torch.arange(n, dtype=torch.int32, device=DEV)

    def step(cache, s, q, k, v, sizes):
        granted = pages_resize(s["refs"], s["tables"], s["lengths"], rows, sizes, page, cache)
        mx4_cache_append(cache, k[:, None], v[:, None], s["tables"], s["lengths"])
        y = cached_attention_step(q, cache, s["tables"], s["lengths"])
        return granted, y, mx4_linear_forward(mx4_quantize(y.flatten(1)), w), mx4_linear_forward(y.flatten(1), w)

    inputs = [(r(n, heads, dim), r(n, kv, dim), r(n, kv, dim), torch.full((n,), t + 1, dtype=torch.int32, device=DEV) + rows * (t > 2))
              for t in range(7)]
    cache, s = make()
    eager = [[t.clone() for t in step(cache, s, *i)] for i in inputs]
    cache, s = make()
    held = [t.clone() for t in inputs[0]]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*make(), *held)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(cache, s, *held)
    for i, ref in zip(inputs, eager):
        for a, b in zip(held, i):
            a.copy_(b)
        graph.replay()
        mx4_linear_forward(torch.randn(70, 256, device=DEV), w)  # eager work of the same kernels
        torch.cuda.synchronize()
        for a, b in zip(outs, ref):
            assert torch.equal(a, b)


def test_other_stream_and_two_at_once():
    """Calls on two streams at a time have workspaces of their own."""
    call, _, q = attention_case(DEV, [1, 1], [4000, 2500], 8, 2, 128, 16, torch.bfloat16, False)
    base = cached_attention_step(q, call["cache"], call["tables"], call["lengths"])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(cached_attention_step(q, call["cache"], call["tables"], call["lengths"]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, base) for y in got)


@pytest.mark.parametrize("n", [1, 150])
@pytest.mark.parametrize("scale", [0.0, -0.3, 5.0])
def test_attention_scales(n, scale):
    """Any scale: 0 weighs every token alike, a negative one turns the order about, a large one picks one token."""
    call, held, q = attention_case(DEV, [n], [45], 2, 1, 64, 16, torch.float32, False)
    y = cached_attention_forward(**call, scale=scale)[0]
    for h in range(2):
        see = torch.arange(n + 45)[None] <= (torch.arange(n) + 45)[:, None]
        ref, mag, big = ora.attend(q[:, h], held[0][0][:, 0], held[0][1][:, 0], see, scale)
        within(y[:, h], ref, attention_bound(torch.float32, 64, n + 45, ref, mag, big), f"scale {scale}")
