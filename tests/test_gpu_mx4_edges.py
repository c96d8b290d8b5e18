"""The 4-bit operators where they can go wrong: numbers that are none, the ends of the scales, many ragged sequences, graphs."""

import pytest
import torch

from oracle import mx4 as ora
from sparseflow_amd.Kernels.cached_attention import MX4Cache, cached_attention_forward, cached_attention_step, mx4_cache_append
from sparseflow_amd.Kernels.mx4 import mx4_linear_forward, mx4_quantize
from sparseflow_amd.Kernels.pages import pages_compact, pages_copy, pages_fork, pages_resize
from tests.gpu_helpers import DEV, announce
from tests.mx4_checks import attention_bound, attention_case, check_attention, check_linear, within
from tests.pages_checks import start

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("m,n", [(3, 150), (40, 150), (40, 2100), (70, 150), (150, 150), (300, 8200)])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_infinities(m, n, dtype):
    """inf times a weight is an infinity of the weight's sign; in float32 and f16, which are taken apart, too."""
    announce(f"linear infinities {m} {n} {dtype}")
    g = torch.Generator().manual_seed(5)
    w = torch.randn(n, 70, generator=g)
    # (At least 0.3 where a block's largest is below 8, whose smallest step is half of one: no weight becomes 0.)
    w = (w.sign() * (w.abs().clamp(max=5) + 0.3)).to(DEV)
    q = mx4_quantize(w)
    values = ora.values(*q, 70)
    assert bool((values != 0).all())
    x = torch.randn(m, 70, generator=g).to(dtype).to(DEV)
    clean = mx4_linear_forward(x, q)
    x[0, 3], x[1, 69] = float("inf"), float("-inf")
    y = mx4_linear_forward(x, q).cpu().double()
    assert torch.equal(y[0], values[:, 3].sign() * float("inf")) and torch.equal(y[1], -values[:, 69].sign() * float("inf"))
    assert torch.equal(y[2:], clean[2:].cpu().double())
    x[0, 4], x[1, 0] = float("inf"), float("nan")
    y = mx4_linear_forward(x, q).cpu()
    split = values[:, 3].sign() != values[:, 4].sign()
    assert torch.isnan(y[0][split]).all() and torch.isinf(y[0][~split]).all() and torch.isnan(y[1]).all()


@pytest.mark.parametrize("m", [33, 64, 65, 100, 128, 200])
@pytest.mark.parametrize("k,n", [(70, 40), (640, 40), (96, 2100), (700, 10300)])
@pytest.mark.parametrize("dtype", TYPES)
def test_linear_groups_of_stages(m, k, n, dtype):
    """Fewer stages than groups, ends of stages, both sides of the rules on rows and columns."""
    check_linear(DEV, m, k, n, dtype, bias=True)


@pytest.mark.parametrize("n", [3, 150])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_nan_behind_the_mask(n, dtype):
    announce(f"attention nan {n} {dtype}")
    call, held, q = attention_case(DEV, [n], [45], 2, 1, 64, 16, dtype, False)
    t = 45 + n // 2
    page, row = int(call["tables"][0, t // 16]), t % 16
    see = torch.arange(n + 45)[None] <= (torch.arange(n) + 45)[:, None]
    for name in ("v_scales", "k_scales"):
        cache = MX4Cache(*(x.clone() for x in call["cache"]))
        getattr(cache, name)[page, 0, row, 1] = 255
        y = cached_attention_forward(**{**call, "cache": cache})[0]
        for h in range(2):
            ref, mag, big = ora.attend(q[:, h], held[0][0][:, 0], held[0][1][:, 0], see, 64 ** -0.5)
            bound = attention_bound(dtype, 64, n + 45, ref, mag, big)
            within(y[:n // 2, h], ref[:n // 2], bound[:n // 2], name)
            if name == "v_scales":
                within(y[n // 2:, h, :32], ref[n // 2:, :32], bound[n // 2:, :32], name)
                assert torch.isnan(y[n // 2:, h, 32:]).all()
            else:
                assert torch.isnan(y[n // 2:, h]).all()


@pytest.mark.parametrize("n", [1, 150])
@pytest.mark.parametrize("byte", [0, 1, 126, 250, 252, 253])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_scales_at_the_ends(n, byte, dtype):
    """Values whose scales are the format's ends, in one token and in all."""
    announce(f"attention far {n} {byte} {dtype}")
    call, held, q = attention_case(DEV, [n], [40], 2, 1, 64, 16, dtype, False)
    see = torch.arange(n + 40)[None] <= (torch.arange(n) + 40)[:, None]
    for rows in ([7], list(range(n + 40))):
        cache = MX4Cache(*(x.clone() for x in call["cache"]))
        for t in rows:
            cache.v_scales[int(call["tables"][0, t // 16]), 0, t % 16, 1] = byte
        v = torch.stack([ora.values(cache.v[int(call["tables"][0, t // 16]), 0, t % 16],
                                    cache.v_scales[int(call["tables"][0, t // 16]), 0, t % 16], 64) for t in range(n + 40)])
        v = v.float().double()  # (a code of 6 with byte 253 is past float32)
        y = cached_attention_forward(**{**call, "cache": cache})[0]
        for h in range(2):
            ref, mag, big = ora.attend(q[:, h], held[0][0][:, 0], v, see, 64 ** -0.5)
            # (Weights of 2^-30 and less times the smallest values: products below float32's normal numbers, 2^-126, are lost.)
            bound = attention_bound(dtype, 64, n + 40, ref, mag, big) + (n + 40) * 2.0 ** -96
            bound = torch.where(torch.isfinite(ref), bound, 0.0)  # (what is none has to be the same one)
            within(y[:, h], ref, bound, f"{byte} {len(rows)}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_steps_of_many_ragged_sequences(dtype):
    announce(f"many ragged {dtype}")
    g = torch.Generator().manual_seed(9)
    old = [int(v) for v in torch.randint(0, 50, (300,), generator=g)]
    check_attention(DEV, [1] * 300, old, 2, 1, 64, 16, dtype, step=True)


@pytest.mark.parametrize("heads,kv", [(4, 2), (8, 1)])
def test_steps_whose_shares_cut_sequences(heads, kv):
    """Long and empty sequences side by side: shares of tokens end inside sequences, and hold several."""
    announce(f"cut shares {heads} {kv}")
    old = [0, 3000, 0, 1, 77, 1500, 0, 64, 63, 2100, 5]
    check_attention(DEV, [1] * len(old), old, heads, kv, 64, 32, torch.bfloat16, step=True)
    check_attention(DEV, [3, 0, 1, 2, 5, 0, 2, 1, 1, 4, 0], old, heads, kv, 64, 32, torch.float32)


def test_longest_length_given():
    """max_len over the longest changes nothing."""
    for dtype, new in ((torch.bfloat16, [3, 40, 1]), (torch.float32, [130, 2, 70])):
        call, _, _ = attention_case(DEV, new, [20, 0, 90], 4, 2, 64, 16, dtype, True)
        y = cached_attention_forward(**call)
        for longest in (None, max(new), sum(new), 10 ** 9):
            got = cached_attention_forward(**{**call, "max_len": longest})
            assert float((got.float() - y.float()).norm() / y.float().norm()) < 2 ** -7


def test_outputs_that_share_memory_are_refused():
    call, _, q = attention_case(DEV, [2, 2], [9, 5], 2, 1, 64, 16, torch.float32, False)
    flat = torch.zeros(2 * q.numel(), device=DEV)
    x = flat[:q.numel()].view(call["q"].shape)
    with pytest.raises(ValueError):
        cached_attention_forward(**{**call, "q": x}, out=flat[64:64 + q.numel()].view(call["q"].shape))
    x = torch.zeros(4, 64, device=DEV)
    w = mx4_quantize(torch.randn(64, 64, device=DEV))
    with pytest.raises(ValueError):
        mx4_linear_forward(x, w, out=x)
    codes = torch.zeros(8, 32, dtype=torch.uint8, device=DEV)
    with pytest.raises(ValueError):
        mx4_quantize(x, out=(codes[:4], codes[3, :8].view(4, 2)))
    k = torch.zeros(2, 2, 1, 64, device=DEV)
    cache = MX4Cache(*(t.clone() for t in call["cache"]))
    with pytest.raises(ValueError):
        mx4_cache_append(cache._replace(v=cache.k), k, k, call["tables"], call["lengths"])
    s = start(DEV, pages=6, rows=3, width=2, page=4)
    rows = torch.tensor([0], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        pages_resize(s["refs"], s["tables"], s["lengths"], s["lengths"][:1], rows, 4, s["pools"])
    with pytest.raises(ValueError):
        pages_copy([s["pools"][0], s["pools"][0]], rows, rows)


def test_two_graphs_have_workspaces_of_their_own():
    """Steps of two batches, captured apart and replayed in turn on two streams at once."""
    calls = [attention_case(DEV, [1, 1], old, 8, 2, 128, 16, torch.bfloat16, False, seed=i)[0]
             for i, old in enumerate(([4000, 2500], [100, 3300]))]
    run = lambda c: cached_attention_forward(**c)  # noqa: E731
    base = [run(c) for c in calls]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        [run(c) for c in calls]
    torch.cuda.current_stream().wait_stream(stream)
    graphs, outs = [], []
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(c))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        [o.zero_() for o in outs]
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        run(calls[0])
        torch.cuda.synchronize()
        assert all(torch.equal(o, b) for o, b in zip(outs, base))


def test_pages_of_nothing():
    """No requests, no pages, no rows."""
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    s = start(DEV, pages=6, rows=3, width=2, page=4)
    none = ints()
    assert pages_resize(s["refs"], s["tables"], s["lengths"], none, none, 4, s["pools"]).shape == (0,)
    assert pages_fork(s["refs"], s["tables"], s["lengths"], none, none, 4, s["pools"]).shape == (0,)
    assert pages_compact(s["refs"], s["tables"], s["pools"]).tolist() == [0]
    pages_copy(s["pools"], none, none)
    for pages, rows in ((0, 3), (6, 0)):
        s = start(DEV, pages=pages, rows=rows, width=2, page=4)
        got = pages_resize(s["refs"], s["tables"], s["lengths"], ints(0, 1), ints(3, 0), 4, s["pools"])
        assert got.tolist() == [0, int(rows > 0)]
        assert pages_fork(s["refs"], s["tables"], s["lengths"], ints(0), ints(1), 4, s["pools"]).tolist() == [int(rows > 0)]
        assert pages_compact(s["refs"], s["tables"], s["pools"]).tolist() == [0]


def test_same_row_twice_in_a_call():
    """The first request of a row counts, on the device as on the host."""
    ints = lambda dev, *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    got = []
    for dev in (DEV, torch.device("cpu")):
        s = start(dev, pages=9, rows=4, width=3, page=4)
        a = pages_resize(s["refs"], s["tables"], s["lengths"], ints(dev, 1, 1, 2), ints(dev, 6, 9, 4), 4, s["pools"])
        b = pages_fork(s["refs"], s["tables"], s["lengths"], ints(dev, 1, 2, 1), ints(dev, 3, 3, 0), 4, s["pools"])
        got.append([t.tolist() for t in (a, b, s["refs"], s["tables"], s["lengths"])])
    assert got[0] == got[1]


def test_steps_of_sequences_that_share_a_slot():
    """Two queries of one row see the same tokens."""
    call, _, q = attention_case(DEV, [1, 1], [40, 7], 4, 2, 64, 16, torch.float16, False)
    q = call["q"][:, 0]
    slots = torch.tensor([1, 0, 1, 1], dtype=torch.int32, device=DEV)
    y = cached_attention_step(q[[1, 0, 1, 0]].contiguous(), call["cache"], call["tables"], call["lengths"], slots=slots)
    base = cached_attention_step(q, call["cache"], call["tables"], call["lengths"])
    assert torch.equal(y[0], base[1]) and torch.equal(y[1], base[0]) and torch.equal(y[2], base[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("four", [False, True], ids=["floats", "4-bit"])
@pytest.mark.parametrize("shape", [(300, 512, 2100), (1100, 256, 1290), (1000, 100, 2561), (3500, 192, 3601), (3333, 70, 4100), (3585, 384, 3600)], ids=str)
def test_linear_tiles_of_every_size(shape, dtype, four):
    """Rows and columns that end inside a tile, in tiles of 64, 128 and 256, few stages and many."""
    announce(f"tiles {shape} {dtype} {four}")
    m, k, n = shape
    check_linear(DEV, m, k, n, dtype, bias=n % 2 == 1, four=four)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(5, 4100, 30), (16, 8200, 40), (64, 4096, 300), (260, 600, 250), (2000, 4224, 50)], ids=str)
def test_linear_pieces(shape, dtype):
    """Few pieces of y, K over many wavefronts: ends of K and of the pieces."""
    m, k, n = shape
    for four in (False, True):
        check_linear(DEV, m, k, n, dtype, bias=True, four=four)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 200])
def test_prompts_in_parts_of_their_tokens(dim, dtype):
    """Few tiles after long contexts: parts joined, among them parts that see nothing, and a sequence without rows."""
    announce(f"prompt parts {dim} {dtype}")
    check_attention(DEV, [60, 0, 130, 1], [2500, 10, 300, 0], 4, 2, dim, 64, dtype)
