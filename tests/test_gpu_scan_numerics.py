"""The scan of prompts where its numbers can go wrong: operands of its products,
long decays, results and states near the ends of a float's range, values that are
not finite.  Against the 64-bit oracle.

Bounds: a bf16 result is off by 2^-8 of itself, an f16 one by 2^-11, a float32 one by
2^-24.  Inside, operands of the products have 16 bits or more (2^-15 of the magnitude
for two of them in a term; float32: all bits), a float32 sum of n terms is off by n
2^-24 of the terms' magnitudes, and a decay is the exponential of a rounded number
(counted with n)."""

import pytest
import torch

from oracle import state_space as ora
from sparseflow_amd.Kernels.selective_scan import selective_scan_forward, selective_scan_step
from tests.gpu_helpers import DEV, announce

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF_ULP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
INNER = {F32: 0.0, F16: 2.0 ** -15, BF16: 2.0 ** -15}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g).to(dtype)


def _bound(n, ref, magnitude, dtype):
    return ((4 * n + 300) * 2.0 ** -24 + INNER[dtype]) * magnitude + HALF_ULP[dtype] * ref.abs() + 2.0 ** -25


def _within(got, want, bound, what):
    got = got.detach().double().cpu()
    off = (got - want).abs() - bound
    assert bool((off <= 0).all()), f"{what}: {float(off.max()):.3g} over the bound, worst error " \
                                   f"{float((got - want).abs().max()):.3g}"


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,H,P,G,N", [(40, 2, 64, 1, 128), (100, 2, 32, 2, 16), (75, 1, 40, 1, 200), (1500, 2, 32, 1, 64)])
@pytest.mark.parametrize("offset", [0, 1])
def test_outputs_are_rounded_once(dtype, n, H, P, G, N, offset):
    """Where the terms of y cancel, what the products' operands lose shows."""
    announce(f"scan rounded once {dtype} n={n} H={H} P={P} G={G} N={N} offset={offset}")
    g = _gen(n + P + N)
    x, dt = _randn(g, 1, n, H, P, dtype=dtype), _randn(g, 1, n, H, dtype=dtype)
    B = _randn(g, 1, n, G, N + offset, dtype=dtype)[..., offset:]
    C = _randn(g, 1, n, G, N + offset, dtype=dtype)[..., offset:]
    A, h0 = -torch.rand(H, generator=g), _randn(g, 1, H, P, N)
    y, state = selective_scan_forward(*_dev(x, dt, A), *(torch.as_strided(t._base.to(DEV) if offset else t.to(DEV), t.shape,
                                                                          t.stride(), t.storage_offset()) for t in (B, C)),
                                      initial_state=h0.to(DEV))
    ref, h, ym, hm = ora.scan(x[0], dt[0], A, B[0], C[0], None, None, True, h0[0])
    _within(y[0], ref, _bound(n, ref, ym, dtype), "y")
    _within(state[0], h, (4 * n + 300) * 2.0 ** -24 * hm, "state")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("offset", [0, 1])
def test_decays_after_one_large_step(dtype, offset):
    """A step that forgets everything leaves exponents of a million behind it in its
    chunk; the decays of the tokens after it are differences of those."""
    announce(f"scan one large step {dtype} offset={offset}")
    n, H, P, G, N = 64, 2, 32, 1, 32
    g = _gen(50)
    x, B, C = (torch.rand(s, generator=g).to(dtype) for s in ((1, n, H, P + offset), (1, n, G, N), (1, n, G, N)))
    x = x[..., offset:]
    dt = torch.full((1, n, H), 1.0 / 128).to(dtype)
    dt[0, 5], dt[0, 40] = 60000.0, 2000.0
    A = torch.tensor([-16.0, -7.3])
    y, state = selective_scan_forward(torch.as_strided(x._base.to(DEV) if offset else x.to(DEV), x.shape, x.stride(),
                                                       x.storage_offset()), *_dev(dt, A, B, C), dt_softplus=False)
    ref, h, ym, hm = ora.scan(x[0], dt[0], A, B[0], C[0], None, None, False, torch.zeros(H, P, N))
    # (What is over the format's range is infinite; no result is within 2^-12 of its end.)
    over = ref.to(dtype).isinf()
    assert bool(((ref / torch.finfo(dtype).max - 1).abs() > 2.0 ** -12).all())
    assert torch.equal(y[0].isinf().cpu(), over)
    _within(torch.where(over.to(DEV), 0, y[0]), torch.where(over, 0, ref), _bound(n, ref, ym, dtype), "y")
    _within(state[0], h, (4 * n + 300) * 2.0 ** -24 * hm, "state")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [70, 1500])
def test_large_results_with_fast_decay(dtype, n):
    """Terms of 2^40 that a chunk decays by 2^-90: finite, whatever factors the decays
    are taken apart into.  (1500 tokens of one head are cut into segments.)"""
    announce(f"scan large results {dtype} n={n}")
    H, P, G, N = 1, 32, 1, 32
    g = _gen(60)
    x, B, C = ((torch.randn(s, generator=g) * 2.0 ** 12).to(dtype) for s in ((1, n, H, P), (1, n, G, N), (1, n, G, N)))
    dt = torch.full((1, n, H), 2.0).to(dtype)
    A = torch.tensor([-0.98])
    y, state = selective_scan_forward(*_dev(x, dt, A, B, C), dt_softplus=False)
    ref, h, ym, hm = ora.scan(x[0], dt[0], A, B[0], C[0], None, None, False, torch.zeros(H, P, N))
    assert float(ref.abs().max()) > 2.0 ** 38
    _within(y[0], ref, _bound(n, ref, ym, dtype), "y")
    _within(state[0], h, (4 * n + 300) * 2.0 ** -24 * hm, "state")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rate", [-0.02, -0.5, 0.0])
@pytest.mark.parametrize("n", [40, 100])
def test_states_near_the_largest_float(dtype, rate, n):
    announce(f"scan large states {dtype} rate={rate} n={n}")
    H, P, G, N = 2, 32, 1, 32
    g = _gen(61)
    x, dt, B = _randn(g, 1, n, H, P, dtype=dtype), torch.full((1, n, H), 1.0).to(dtype), _randn(g, 1, n, G, N, dtype=dtype)
    C = torch.zeros(1, n, G, N, dtype=dtype)
    A, h0 = torch.full((H,), rate), _randn(g, 1, H, P, N) * 2.0 ** 118
    y, state = selective_scan_forward(*_dev(x, dt, A, B, C), dt_softplus=False, initial_state=h0.to(DEV))
    ref, h, _, hm = ora.scan(x[0], dt[0], A, B[0], C[0], None, None, False, h0[0])
    assert torch.isfinite(state).all() and not y.any()
    _within(state[0], h, (4 * n + 300) * 2.0 ** -24 * hm, "state")


def test_inputs_and_states_near_the_largest_float32():
    """Above 3.39e38 a float32 rounds to infinity in bf16."""
    announce("scan float32 inputs near the largest float")
    n, H, P, G, N, most = 50, 2, 32, 1, 32, 3.4e38
    g = _gen(62)
    x, dt, A = _randn(g, 1, n, H, P), torch.full((1, n, H), 1.0), torch.tensor([-0.1, -3.0])
    B, C = _randn(g, 1, n, G, N), _randn(g, 1, n, G, N)
    x[0, 20, 0, 3], B[0, 20] = most, B[0, 20] * 1e-30
    h0 = _randn(g, 1, H, P, N)
    h0[0, 1, 5, 7], C[0, 0] = most, C[0, 0] * 1e-30
    y, state = selective_scan_forward(*_dev(x, dt, A, B, C), dt_softplus=False, initial_state=h0.to(DEV))
    ref, h, ym, hm = ora.scan(x[0], dt[0], A, B[0], C[0], None, None, False, h0[0])
    ok = ym < 2.0 ** 127
    assert bool(ok[:, 0].all()) and bool(ok[0].all()) and torch.isfinite(y[0].cpu()[ok]).all()
    _within(torch.where(ok, y[0].double().cpu(), ref), ref, _bound(n, ref, ym, F32), "y")
    _within(state[0], h, (4 * n + 300) * 2.0 ** -24 * hm, "state")


def _same_values(got, want, what):
    got = got.detach().double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: {int((torch.isnan(got) != torch.isnan(want)).sum())} NaN"
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), f"{what}: infinities"


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("where", ["x", "B", "C", "state", "several"])
@pytest.mark.parametrize("n,at,step", [(20, 0, 0.25), (100, 77, 0.25), (1500, 300, 0.25), (1500, 300, 4.0)])
def test_infinities_are_those_of_the_recurrence(dtype, where, n, at, step):
    """(1500 tokens of two heads are cut into segments.)"""
    announce(f"scan infinities in {where} {dtype} n={n} step={step}")
    H, P, G, N = 2, 40, 2, 48
    g = _gen(63)
    x = _randn(g, 1, n, H, P, dtype=dtype)
    B, C = ((torch.rand(1, n, G, N, generator=g) + 0.25).to(dtype) for _ in range(2))
    # (1.0: exact in one part, whose other parts are zeros.)
    B[..., ::3], C[..., ::2] = 1.0, 1.0
    dt, A = torch.full((1, n, H), step).to(dtype), torch.tensor([-0.125, -1.0])
    h0, inf = _randn(g, 1, H, P, N), float("inf")
    if where in ("x", "several"):
        x[0, at, 1, 3], x[0, at, 1, 33] = inf, -inf
    if where in ("B", "several"):
        B[0, at, 1, 5] = inf
    if where in ("C", "several"):
        C[0, at, 1, 6] = -inf
    if where == "state":
        h0[0, 1, 2, 4], h0[0, 1, 3] = inf, -inf
    y, state = selective_scan_forward(*_dev(x, dt, A, B, C), dt_softplus=False, initial_state=h0.to(DEV))
    ref, h, ym, hm = ora.scan(x[0], dt[0], A, B[0], C[0], None, None, False, h0[0])
    _same_values(y[0], ref, "y")
    _same_values(state[0], h, "state")
    ok, fine = torch.isfinite(ref), torch.isfinite(h)
    assert bool(ok[:, 0].all()) and not bool(ok[:, 1].all())
    for got, want, bound, keep in ((y[0], ref, _bound(n, ref, ym, dtype), ok),
                                   (state[0], h, (4 * n + 300) * 2.0 ** -24 * hm, fine)):
        _within(torch.where(keep.to(DEV), got, 0), torch.where(keep, want, 0), torch.where(keep, bound, 0), "finite ones")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_large_term_after_a_slow_decay(dtype):
    """2^118 comes in when the chunks before have decayed the state by 2^-17."""
    announce(f"scan large term after slow decay {dtype}")
    n, H, P, G, N = 90, 1, 32, 1, 32
    g = _gen(64)
    x, B = _randn(g, 1, n, H, P, dtype=dtype), _randn(g, 1, n, G, N, dtype=dtype)
    C = (torch.randn(1, n, G, N, generator=g) * 2.0 ** -40).to(dtype)
    x[0, 80] *= 2.0 ** 60
    B[0, 80] *= 2.0 ** 58
    dt, A = torch.ones(1, n, H, dtype=dtype), torch.tensor([-0.1317])
    y, state = selective_scan_forward(*_dev(x, dt, A, B, C), dt_softplus=False)
    ref, h, ym, hm = ora.scan(x[0], dt[0], A, B[0], C[0], None, None, False, torch.zeros(H, P, N))
    _within(y[0], ref, _bound(n, ref, ym, dtype), "y")
    _within(state[0], h, (4 * n + 300) * 2.0 ** -24 * hm, "state")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n", [1, 5])
def test_infinities_token_by_token(dtype, n):
    """Without D an infinite x is not multiplied by a zero one."""
    announce(f"scan infinities token by token {dtype} n={n}")
    H, P, G, N, inf = 2, 40, 1, 48, float("inf")
    g = _gen(65)
    x = _randn(g, 2, n, H, P, dtype=dtype)
    B, C = ((torch.rand(2, n, G, N, generator=g) + 0.25).to(dtype) for _ in range(2))
    dt, A, h0 = torch.full((2, n, H), 0.25).to(dtype), torch.tensor([-0.125, -1.0]), _randn(g, 2, H, P, N)
    x[0, 0, 1, 3], x[1, n - 1, 0, 39] = inf, -inf
    y, state = selective_scan_forward(*_dev(x, dt, A, B, C), dt_softplus=False, initial_state=h0.to(DEV))
    for b in range(2):
        ref, h, _, _ = ora.scan(x[b], dt[b], A, B[b], C[b], None, None, False, h0[b])
        assert not torch.isnan(ref).any()
        _same_values(y[b], ref, "y")
        _same_values(state[b], h, "state")
    if n == 1:
        pool = h0.to(DEV)
        step = selective_scan_step(pool, *_dev(x[:, 0], dt[:, 0], A, B[:, 0], C[:, 0]), dt_softplus=False)
        assert torch.equal(step, y[:, 0]) and torch.equal(pool, state)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,rate", [(20, -0.3), (37, -0.05), (64, -1.0), (300, -0.02), (300, -0.4), (1500, -0.1)])
def test_states_to_a_float32s_last_bits(dtype, n, rate):
    """A term has a handful of roundings (step, exponential, their product with x, parts,
    sums of eight terms and of the chunks behind it), each of 2^-24 of it at most and of
    either sign: 2^-22 of the 2-norm is four of them in a row.  (An exponent that is
    rounded as one float costs 2^-20 from 16 on.)"""
    announce(f"scan states to the last bits {dtype} n={n} rate={rate}")
    H, P, G, N = 3, 32, 1, 64
    g = _gen(66)
    x, B, C = _randn(g, 1, n, H, P, dtype=dtype), _randn(g, 1, n, G, N, dtype=dtype), _randn(g, 1, n, G, N, dtype=dtype)
    dt, A = (torch.rand(1, n, H, generator=g) + 0.5).to(dtype), torch.tensor([rate, rate * 1.7, rate * 0.6])
    h0 = _randn(g, 1, H, P, N)
    _, state = selective_scan_forward(*_dev(x, dt, A, B, C), dt_softplus=False, initial_state=h0.to(DEV))
    _, h, _, _ = ora.scan(x[0], dt[0], A, B[0], C[0], None, None, False, h0[0])
    for k in range(H):
        off = float((state[0, k].double().cpu() - h[k]).norm() / h[k].norm())
        assert off <= 2.0 ** -22, f"head {k}: 2-norm off by {off * 2 ** 22:.2f} of what is allowed"
