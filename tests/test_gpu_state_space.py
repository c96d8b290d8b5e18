"""The state space operators (causal convolution, selective scan, block norm)
on the GPU against the 64-bit oracle, for prompts and single tokens.

Tolerances come from the formats.  A result rounded to a format with p
significant bits is off by at most 2^-p of itself (bf16 2^-8, f16 2^-11); float32
sums of n terms are off by n 2^-24 of the sum of the terms' magnitudes.  The scan
of bf16 inputs may round its products' operands to bf16 once more (2^-8 of the
magnitude); its states are float32 whatever the inputs.
"""

import pytest
import torch

from oracle import state_space as ora
from sparseflow_amd import _lib
from sparseflow_amd.Kernels.block_norm import block_norm_forward
from sparseflow_amd.Kernels.causal_conv1d import causal_conv1d_forward, causal_conv1d_step
from sparseflow_amd.Kernels.selective_scan import selective_scan_forward, selective_scan_step
from tests.gpu_helpers import DEV, announce, native_loaded

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF_ULP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
# Of the magnitude, by the roundings within the scan's products.
INNER = {F32: 0.0, F16: 2.0 ** -15, BF16: 2.0 ** -8}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=F32, gain=1.0):
    return (torch.randn(shape, generator=g) * gain).to(dtype)


def _within(got, want, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, what
    off = (got - want).abs() - bound
    assert bool((off <= 0).all()), f"{what}: {float(off.max()):.3g} over the bound, worst error " \
                                   f"{float((got - want).abs().max()):.3g}"


def _near(got, want, rel, what):
    got = got.detach().double().cpu()
    off = float((got - want).norm() / want.norm().clamp(min=1e-300))
    assert off <= rel, f"{what}: 2-norm off by {off:.3g}, {rel:.3g} allowed"


# ---- causal convolution -------------------------------------------------------


def _conv_check(y, state, x, w, bias, act, before, dtype, what):
    ref, ref_state, mag = ora.conv1d(x.cpu(), w.cpu(), None if bias is None else bias.cpu(), act, before.cpu())
    # K + 1 float32 roundings, silu's own few, the result's.
    n = w.shape[1] + 8
    _within(y, ref, n * 2.0 ** -24 * (1 + mag) * 1.2 + HALF_ULP[dtype] * ref.abs() + 2.0 ** -25, what)
    assert torch.equal(state.double().cpu(), ref_state), f"{what}: state"


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,c,k", [(1, 8, 4), (2, 5, 4), (3, 64, 4), (16, 37, 2), (17, 96, 3), (65, 129, 8),
                                   (200, 256, 4), (33, 12, 1), (40, 24, 5), (41, 16, 6), (18, 40, 7)])
@pytest.mark.parametrize("initial", [False, True])
def test_conv_prompt(dtype, n, c, k, initial):
    announce(f"conv prompt {dtype} n={n} c={c} k={k} initial={initial}")
    g = _gen(n * 1000 + c + k)
    x, w, b = _randn(g, 3, n, c, dtype=dtype), _randn(g, c, k), _randn(g, c)
    before = _randn(g, 3, k - 1, c, dtype=dtype) if initial else torch.zeros(3, k - 1, c, dtype=dtype)
    act = "silu" if c % 2 == 0 else None
    y, state = causal_conv1d_forward(x.to(DEV), w.to(DEV), b.to(DEV), activation=act,
                                     initial_state=before.to(DEV) if initial else None)
    for i in range(3):
        _conv_check(y[i], state[i], x[i], w, b, act, before[i], dtype, f"sequence {i}")
    assert native_loaded()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens", [[0], [5, 0, 1, 2, 40, 0], [0, 0, 100, 17, 16, 15, 3]])
@pytest.mark.parametrize("hint", ["exact", "none", "short"])
def test_conv_packed(dtype, lens, hint):
    announce(f"conv packed {dtype} {lens} max_len {hint}")
    g = _gen(sum(lens) + len(lens))
    c, k = 48, 4
    off = [0]
    for v in lens:
        off.append(off[-1] + v)
    x, w = _randn(g, off[-1], c, dtype=dtype), _randn(g, c, k)
    before = _randn(g, len(lens), k - 1, c, dtype=dtype)
    max_len = {"exact": max(lens), "none": None, "short": 1}[hint]
    y, state = causal_conv1d_forward(x.to(DEV), w.to(DEV), activation="silu", initial_state=before.to(DEV),
                                     offsets=torch.tensor(off, dtype=torch.int32, device=DEV), max_len=max_len)
    for i, v in enumerate(lens):
        _conv_check(y[off[i]:off[i + 1]], state[i], x[off[i]:off[i + 1]], w, None, "silu", before[i], dtype,
                    f"sequence {i} of {v}")


def test_conv_strided_views_pool_in_place_and_step():
    announce("conv views, pool in place, steps")
    g = _gen(5)
    c, k, n, rows = 40, 4, 50, 6
    wide = _randn(g, 2, n, 3 * c, dtype=BF16).to(DEV)
    x = wide[..., c:2 * c]
    w, b = _randn(g, c, k).to(DEV), _randn(g, c).to(DEV)
    pool = _randn(g, rows, k - 1, c, dtype=BF16).to(DEV)
    start = pool.clone()
    slots = torch.tensor([4, 1], dtype=torch.int32, device=DEV)
    y, kept = causal_conv1d_forward(x, w, b, initial_state=pool, final_state=pool, slots=slots)
    assert kept is pool
    for i, s in enumerate((4, 1)):
        _conv_check(y[i], pool[s], x[i], w, b, None, start[s], BF16, f"slot {s}")
    assert torch.equal(pool[[0, 2, 3, 5]], start[[0, 2, 3, 5]])
    # The same prompt token by token, one of three sequences without a row.
    step_pool = start.clone()
    slots3 = torch.tensor([4, -1, 1], dtype=torch.int32, device=DEV)
    for t in range(n):
        xt = torch.stack([x[0, t], x[0, t], x[1, t]])
        yt = causal_conv1d_step(step_pool, xt, w, b, slots=slots3)
        assert torch.equal(yt[0], y[0, t]) and torch.equal(yt[2], y[1, t])
        assert not yt[1].any()
    assert torch.equal(step_pool, pool)
    out_of_pool = torch.tensor([rows, 1, -7], dtype=torch.int32, device=DEV)
    before = step_pool.clone()
    yt = causal_conv1d_step(step_pool, xt, w, b, slots=out_of_pool)
    assert not yt[0].any() and not yt[2].any() and yt[1].any()
    assert torch.equal(step_pool[[0, 2, 3, 4, 5]], before[[0, 2, 3, 4, 5]])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,c", [(1, 13), (6, 37), (90, 1037), (40, 3), (50, 64)])
def test_conv_odd_rows_at_any_address_and_in_place(dtype, n, c):
    announce(f"conv odd rows {dtype} n={n} c={c}")
    g = _gen(n + c)
    k, off = 4, 3
    wide = _randn(g, 2, n, c + off, dtype=dtype).to(DEV)
    x = wide[..., off:]
    w, b = _randn(g, c, k).to(DEV), _randn(g, c).to(DEV)
    pool = torch.zeros(1 + 2 * (k - 1) * c, dtype=dtype, device=DEV)[1:].view(2, k - 1, c)
    pool.copy_(_randn(g, 2, k - 1, c, dtype=dtype))
    start = pool.clone()
    y, kept = causal_conv1d_forward(x, w, b, activation="silu", initial_state=pool, final_state=pool)
    assert kept is pool
    for i in range(2):
        _conv_check(y[i], pool[i], x[i], w, b, "silu", start[i], dtype, f"sequence {i}")
    stepped = start.clone()
    for t in range(min(n, 9)):
        yt = causal_conv1d_step(stepped, x[:, t], w, b, activation="silu")
        assert torch.equal(yt, y[:, t])


# ---- selective scan -----------------------------------------------------------


def _scan_inputs(g, lead, H, P, G, N, dtype):
    # Views of wider rows, as projections leave them.
    xbc = _randn(g, *lead, H * P + 2 * G * N, dtype=dtype)
    x = xbc[..., :H * P].unflatten(-1, (H, P))
    B = xbc[..., H * P:H * P + G * N].unflatten(-1, (G, N))
    C = xbc[..., H * P + G * N:].unflatten(-1, (G, N))
    dt = _randn(g, *lead, H + 3, dtype=dtype)[..., 3:]
    A = -torch.rand(H, generator=g) * 8
    A[0] = 0.0  # a head that forgets nothing
    D, bias = _randn(g, H), torch.rand(H, generator=g) * 4 - 5
    return x, dt, A, B, C, D, bias


def _scan_check(y, state, x, dt, A, B, C, D, bias, softplus, h0, dtype, what):
    ref, h, ym, hm = ora.scan(x, dt, A, B, C, D, bias, softplus, h0)
    # Float32: a term passes through a product per token behind it (and the
    # exponential's argument is rounded), and 256 terms meet in the last sum.
    n = 4 * x.shape[0] + 300
    if x.shape[0]:
        _within(y, ref, (n * 2.0 ** -24 + INNER[dtype]) * ym + HALF_ULP[dtype] * ref.abs() + 2.0 ** -25, f"{what}: y")
        _near(y, ref, {F32: 2.0 ** -17, F16: 2.0 ** -11, BF16: 2.0 ** -8}[dtype], f"{what}: y")
    _within(state, h, n * 2.0 ** -24 * hm + 1e-30, f"{what}: state")
    _near(state, h, 2.0 ** -18, f"{what}: state")


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


def _on_device(t):
    """A view's device copy with the same strides."""
    base = t._base if t._base is not None else t
    return torch.as_strided(base.to(DEV), t.shape, t.stride(), t.storage_offset())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,H,P,G,N", [
    (1, 3, 64, 1, 64), (2, 2, 32, 1, 16), (15, 1, 16, 1, 128), (16, 2, 64, 2, 128), (31, 4, 20, 2, 24),
    (63, 2, 64, 1, 128), (64, 3, 64, 1, 64), (65, 4, 32, 4, 256), (130, 2, 128, 1, 64), (37, 3, 7, 1, 5),
    (200, 2, 100, 2, 130), (129, 1, 1, 1, 1), (257, 6, 48, 3, 80), (90, 2, 160, 1, 33)])
@pytest.mark.parametrize("initial", [False, True])
def test_scan_prompt(dtype, n, H, P, G, N, initial):
    announce(f"scan prompt {dtype} n={n} H={H} P={P} G={G} N={N} initial={initial}")
    g = _gen(n + H * 7 + P * 11 + N * 13)
    x, dt, A, B, C, D, bias = _scan_inputs(g, (2, n), H, P, G, N, dtype)
    h0 = _randn(g, 2, H, P, N) if initial else None
    y, state = selective_scan_forward(_on_device(x), _on_device(dt), A.to(DEV), _on_device(B), _on_device(C), D.to(DEV),
                                      bias.to(DEV), initial_state=None if h0 is None else h0.to(DEV))
    for b in range(2):
        _scan_check(y[b], state[b], x[b], dt[b], A, B[b], C[b], D, bias, True,
                    torch.zeros(H, P, N) if h0 is None else h0[b], dtype, f"sequence {b}")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_scan_long_few_heads_is_split(dtype):
    announce(f"scan long {dtype}")
    n, H, P, G, N = 1111, 2, 32, 1, 32
    g = _gen(3)
    x, dt, A, B, C, D, bias = _scan_inputs(g, (1, n), H, P, G, N, dtype)
    h0 = _randn(g, 1, H, P, N)
    y, state = selective_scan_forward(*_dev(x, dt, A, B, C), initial_state=h0.to(DEV))
    _scan_check(y[0], state[0], x[0], dt[0], A, B[0], C[0], None, None, True, h0[0], dtype, "long")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens", [[0], [0, 3, 0, 70, 1, 64, 0], [300, 0, 65, 129, 2]])
@pytest.mark.parametrize("hint", ["exact", "none", "short"])
def test_scan_packed(dtype, lens, hint):
    announce(f"scan packed {dtype} {lens} max_len {hint}")
    H, P, G, N = 4, 32, 2, 64
    g = _gen(sum(lens) + 1)
    off = [0]
    for v in lens:
        off.append(off[-1] + v)
    x, dt, A, B, C, D, bias = _scan_inputs(g, (off[-1],), H, P, G, N, dtype)
    rows = len(lens) + 3
    pool = _randn(g, rows, H, P, N)
    slots = torch.randperm(rows, generator=g)[:len(lens)].to(torch.int32)
    dev_pool = pool.to(DEV)
    max_len = {"exact": max(lens), "none": None, "short": 1}[hint]
    y, kept = selective_scan_forward(*_dev(x, dt, A, B, C, D, bias), initial_state=dev_pool, final_state=dev_pool,
                                     slots=slots.to(DEV), offsets=torch.tensor(off, dtype=torch.int32, device=DEV),
                                     max_len=max_len)
    assert kept is dev_pool
    for i, v in enumerate(lens):
        s, at = int(slots[i]), slice(off[i], off[i + 1])
        _scan_check(y[at], dev_pool[s], x[at], dt[at], A, B[at], C[at], D, bias, True, pool[s], dtype,
                    f"sequence {i} of {v}")
    rest = [r for r in range(rows) if r not in slots.tolist()]
    assert torch.equal(dev_pool[rest].cpu(), pool[rest])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens,P,N", [([1200, 0, 31, 700], 64, 128), ([0, 999], 40, 256)])
def test_scan_packed_is_split_with_states_at_any_address(dtype, lens, P, N):
    announce(f"scan split {dtype} {lens} P={P} N={N}")
    H, G = 2, 1
    g = _gen(sum(lens) + P)
    off = [0]
    for v in lens:
        off.append(off[-1] + v)
    x, dt, A, B, C, D, bias = _scan_inputs(g, (off[-1],), H, P, G, N, dtype)
    h0 = _randn(g, len(lens), H, P, N)
    # (States that begin one float after a multiple of 16 bytes.)
    kept, before = (torch.zeros(h0.numel() + 1, device=DEV)[1:].view(h0.shape) for _ in range(2))
    before.copy_(h0)
    y, state = selective_scan_forward(*_dev(x, dt, A, B, C, D, bias), initial_state=before, final_state=kept,
                                      offsets=torch.tensor(off, dtype=torch.int32, device=DEV), max_len=max(lens))
    assert state is kept and torch.equal(before.cpu(), h0)
    for i, v in enumerate(lens):
        at = slice(off[i], off[i + 1])
        _scan_check(y[at], kept[i], x[at], dt[at], A, B[at], C[at], D, bias, True, h0[i], dtype, f"sequence {i} of {v}")


def test_scan_workspace_is_reused_or_refused():
    g = _gen(8)
    x, dt, A, B, C, D, bias = _dev(*_scan_inputs(g, (1, 600), 1, 32, 1, 32, F32))
    ws = torch.empty(1 << 24, dtype=torch.uint8, device=DEV)
    want = selective_scan_forward(x, dt, A, B, C, D, bias)
    got = selective_scan_forward(x, dt, A, B, C, D, bias, workspace=ws)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(_lib.SparseFlowLibError, match="16 bytes"):
        selective_scan_forward(x, dt, A, B, C, D, bias, workspace=ws[1:])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,P,G,N", [(3, 64, 1, 64), (8, 64, 1, 128), (4, 20, 2, 24), (3, 7, 1, 5), (2, 128, 1, 256),
                                     (4, 33, 4, 100)])
def test_scan_step(dtype, H, P, G, N):
    announce(f"scan step {dtype} H={H} P={P} G={G} N={N}")
    g = _gen(H + P + N)
    batch, rows = 5, 9
    x, dt, A, B, C, D, bias = _scan_inputs(g, (batch,), H, P, G, N, dtype)
    pool = _randn(g, rows, H, P, N)
    slots = [7, -1, 0, 8, rows]
    dev_pool = pool.to(DEV)
    y = selective_scan_step(dev_pool, _on_device(x), _on_device(dt), A.to(DEV), _on_device(B), _on_device(C), D.to(DEV),
                            bias.to(DEV), slots=torch.tensor(slots, dtype=torch.int32, device=DEV))
    for b, s in enumerate(slots):
        if not 0 <= s < rows:
            assert not y[b].any()
            continue
        ref, h, ym, hm = ora.scan(x[b:b + 1], dt[b:b + 1], A, B[b:b + 1], C[b:b + 1], D, bias, True, pool[s])
        _within(y[b], ref[0], 300 * 2.0 ** -24 * ym[0] + HALF_ULP[dtype] * ref[0].abs() + 2.0 ** -25, "y")
        _within(dev_pool[s], h, 16 * 2.0 ** -24 * hm, "state")
    rest = [r for r in range(rows) if r not in slots]
    assert torch.equal(dev_pool[rest].cpu(), pool[rest])


def test_scan_steps_continue_a_prompt():
    announce("prompt then steps")
    H, P, G, N, n = 4, 32, 1, 64, 70
    g = _gen(12)
    x, dt, A, B, C, D, bias = _scan_inputs(g, (2, n), H, P, G, N, F32)
    dx, ddt, dA, dB, dC, dD, dbias = _dev(x, dt, A, B, C, D, bias)
    whole, last = selective_scan_forward(dx, ddt, dA, dB, dC, dD, dbias)
    cut = 61
    y, state = selective_scan_forward(dx[:, :cut], ddt[:, :cut], dA, dB[:, :cut], dC[:, :cut], dD, dbias)
    for t in range(cut, n):
        yt = selective_scan_step(state, dx[:, t], ddt[:, t], dA, dB[:, t], dC[:, t], dD, dbias)
        assert torch.allclose(yt, whole[:, t], rtol=1e-5, atol=1e-5)
    assert torch.allclose(state, last, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("where", ["x", "B", "C", "dt"])
def test_scan_bad_values_reach_later_tokens_only(dtype, bad, where):
    """Causality holds for values that are not finite: what they touch is as in
    the recurrence, everything before as without them."""
    announce(f"scan {bad} in {where} {dtype}")
    H, P, G, N, n, at = 2, 32, 2, 64, 150, 77
    g = _gen(21)
    x, dt, A, B, C, D, bias = (t.clone() for t in _scan_inputs(g, (1, n), H, P, G, N, dtype))
    clean, _ = selective_scan_forward(*_dev(x, dt, A, B, C, D, bias))
    {"x": x, "B": B, "C": C, "dt": dt}[where][0, at, 1 if where != "dt" else slice(1, 2)] = bad
    y, state = selective_scan_forward(*_dev(x, dt, A, B, C, D, bias))
    assert torch.equal(y[:, :, 0], clean[:, :, 0])  # the other head (and group)
    assert torch.isfinite(y[:, :at]).all()
    ref, h, ym, _ = ora.scan(x[0], dt[0], A, B[0], C[0], D, bias, True, torch.zeros(H, P, N))
    _within(y[0, :at], ref[:at], (1000 * 2.0 ** -24 + INNER[dtype]) * ym[:at] + HALF_ULP[dtype] * ref[:at].abs() + 2.0 ** -25,
            "before")
    got = y[0].double().cpu()
    assert torch.equal(torch.isfinite(got), torch.isfinite(ref.to(dtype).double()))
    if where == "C":
        assert torch.isfinite(got[at + 1:]).all() and torch.isfinite(state).all()
    assert torch.equal(torch.isfinite(state[0].double().cpu()), torch.isfinite(h))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,H,P,G,N", [(5, 3, 64, 1, 64), (75, 4, 64, 2, 128), (700, 2, 40, 1, 96), (40, 2, 36, 1, 20)])
def test_scan_rows_at_any_address(dtype, n, H, P, G, N):
    announce(f"scan odd rows {dtype} n={n} H={H} P={P} G={G} N={N}")
    g = _gen(n + P)
    _, dt, A, _, _, D, bias = _scan_inputs(g, (2, n), H, P, G, N, dtype)
    row = _randn(g, 2, n, 1 + H * P + 2 * G * N, dtype=dtype)  # an odd number of elements from row to row
    x = row[..., 1:1 + H * P].unflatten(-1, (H, P))
    B, C = (row[..., 1 + H * P + i * G * N:1 + H * P + (i + 1) * G * N].unflatten(-1, (G, N)) for i in range(2))
    h0 = _randn(g, 2, H, P, N)
    out = torch.zeros(2, n, H * P + 3, dtype=dtype, device=DEV)[..., 1:1 + H * P].unflatten(-1, (H, P))
    y, state = selective_scan_forward(_on_device(x), _on_device(dt), A.to(DEV), _on_device(B), _on_device(C), D.to(DEV),
                                      bias.to(DEV), initial_state=h0.to(DEV), out=out)
    assert y is out and not out._base[..., 0].any() and not out._base[..., 1 + H * P:].any()
    for b in range(2):
        _scan_check(y[b], state[b], x[b], dt[b], A, B[b], C[b], D, bias, True, h0[b], dtype, f"sequence {b}")


def test_scan_without_softplus_and_strides_of_its_own():
    announce("scan no softplus, head-major views")
    H, P, G, N, n = 4, 32, 2, 32, 100
    g = _gen(31)
    x, dt, A, B, C, D, _ = _scan_inputs(g, (2, n), H, P, G, N, F32)
    dt = dt.abs() * 0.05
    hx = x.permute(0, 2, 1, 3).contiguous().to(DEV).permute(0, 2, 1, 3)  # [b, n, H, P] over head-major memory
    hdt = dt.permute(2, 0, 1).contiguous().to(DEV).permute(1, 2, 0)
    hB = B.permute(1, 0, 2, 3).contiguous().to(DEV).permute(1, 0, 2, 3)
    out = torch.empty(H, 2, n, P, device=DEV).permute(1, 2, 0, 3)
    y, state = selective_scan_forward(hx, hdt, A.to(DEV), hB, C.to(DEV), D.to(DEV), dt_softplus=False, out=out)
    assert y is out
    for b in range(2):
        _scan_check(y[b], state[b], x[b], dt[b], A, B[b], C[b], D, None, False, torch.zeros(H, P, N), F32, f"{b}")


# ---- block norm ---------------------------------------------------------------


@pytest.mark.parametrize("dtype,res", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("rows,dim", [(1, 64), (5, 37), (3, 1), (4, 384), (7, 1000), (3, 2048), (2, 4097), (2, 8192),
                                      (1, 16384), (130, 96)])
@pytest.mark.parametrize("form", ["pre", "gated", "between", "after", "plain"])
def test_block_norm(dtype, res, rows, dim, form):
    announce(f"norm {dtype} {res} {rows}x{dim} {form}")
    g = _gen(rows + dim)
    x, gate = _randn(g, rows, dim, dtype=dtype), _randn(g, rows, dim, dtype=dtype, gain=2.0)
    post, pre, scale = torch.rand(dim, generator=g) + 0.5, torch.rand(dim, generator=g) + 0.5, _randn(g, dim)
    residual = _randn(g, rows, dim, dtype=res)
    kw = {"pre": dict(pre_weight=pre, residual=residual),
          "gated": dict(gate=gate, gate_first=True, post_weight=post, group_size=dim // 4 if dim % 4 == 0 else dim),
          "between": dict(gate=gate, post_weight=post, residual=residual, scale=scale, pre_weight=pre,
                          group_size=dim // 8 if dim % 8 == 0 else dim, activation="sigmoid"),
          "after": dict(post_weight=post, residual=residual, scale=0.25),
          "plain": dict(gate=gate, activation=None, residual=residual)}[form]
    eps = 1e-5
    r, h = block_norm_forward(x.to(DEV), eps=eps,
                              **{k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in kw.items()})
    rr, hh, mag = ora.block_norm(x, kw.get("gate"), kw.get("activation", "silu"), kw.get("gate_first", False),
                                 kw.get("post_weight"), kw.get("group_size", dim), kw.get("residual"),
                                 kw.get("scale"), kw.get("pre_weight"), eps)
    r_type = res if "residual" in kw else dtype
    assert r.dtype == r_type and (h is None) == (hh is None)
    # A few float32 roundings; a sum of squares of n terms adds in a tree (of at most 64 in a row).
    f = 100 * 2.0 ** -24
    _within(r, rr, f * mag + HALF_ULP[r_type] * rr.abs() + 2.0 ** -25, "r")
    if h is not None:
        rms = torch.sqrt(rr.square().mean(-1, keepdim=True) + eps)
        _within(h, hh, 2 * f * (mag / rms * pre + hh.abs()) + HALF_ULP[dtype] * hh.abs() + 2.0 ** -25, "h")


@pytest.mark.parametrize("dtype,res", [(F32, F32), (F16, F16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("rows,dim", [(3, 64), (2, 1024), (5, 104)])
def test_block_norm_rows_at_any_address(dtype, res, rows, dim):
    announce(f"norm odd rows {dtype} {res} {rows}x{dim}")
    g = _gen(rows + dim)
    x, gate = (_randn(g, rows, dim + 1, dtype=dtype).to(DEV)[:, 1:] for _ in range(2))
    residual = _randn(g, rows, dim + 3, dtype=res).to(DEV)[:, 3:]
    w, pre = torch.rand(dim, generator=g) + 0.5, torch.rand(dim, generator=g) + 0.5
    kw = dict(post_weight=w.to(DEV), group_size=dim // 8, pre_weight=pre.to(DEV))
    r, h = block_norm_forward(x, gate, residual=residual, **kw)
    r2, h2 = block_norm_forward(x.contiguous(), gate.contiguous(), residual=residual.contiguous(), **kw)
    assert torch.equal(r, r2) and torch.equal(h, h2)


def test_block_norm_strides_broadcasts_and_in_place():
    announce("norm strides, broadcast gate, in place")
    g = _gen(8)
    b, n, dim = 3, 17, 128
    wide = _randn(g, b, n + 2, 2 * dim, dtype=BF16).to(DEV)
    x = wide[:, 1:n + 1, dim:]
    gate = _randn(g, b, 1, dim, dtype=BF16).to(DEV)
    residual = _randn(g, b, n, dim).to(DEV)
    post, pre = torch.rand(dim, generator=g).to(DEV), torch.rand(dim, generator=g).to(DEV)
    want_r, want_h, mag = ora.block_norm(x.cpu(), gate.cpu(), "silu", False, post.cpu(), dim, residual.cpu(), 0.5,
                                         pre.cpu(), 1e-6)
    before = wide.clone()
    r, h = block_norm_forward(x, gate=gate, post_weight=post, residual=residual, scale=0.5, pre_weight=pre, out=x,
                              residual_out=residual)
    assert r is residual and h is x
    _within(r, want_r, 200 * 2.0 ** -24 * mag + 2.0 ** -25, "r")
    _within(h, want_h, 2.0 ** -8 * want_h.abs() + 1e-4, "h")
    before[:, 1:n + 1, dim:] = x
    assert torch.equal(before, wide)  # nothing else was written


def test_block_norm_zero_rows_and_bad_values_stay_in_their_row():
    announce("norm zero rows, bad rows")
    g = _gen(9)
    x = _randn(g, 6, 300)
    x[2] = 0
    x[4, 17] = float("nan")
    x[5, 3] = float("inf")
    w = torch.ones(300)
    r, h = block_norm_forward(x.to(DEV), pre_weight=w.to(DEV))
    assert torch.equal(h[2].cpu(), torch.zeros(300))
    assert torch.isfinite(h[:4]).all() and torch.isnan(h[4]).all()
    assert torch.isnan(h[5, 3]) and not h[5, :3].any()


# ---- streams and graphs ---------------------------------------------------------


def test_operators_run_on_the_current_stream_and_replay_in_a_graph():
    announce("streams and graph")
    H, P, G, N, n, c, k = 4, 32, 1, 64, 100, 128, 4
    g = _gen(40)
    x, dt, A, B, C, D, bias = _dev(*_scan_inputs(g, (2, n), H, P, G, N, BF16))
    w, pre = _randn(g, c, k).to(DEV), torch.rand(c, generator=g).to(DEV)
    xc = _randn(g, 2, n, c, dtype=BF16).to(DEV)

    def all_of_them():
        u, cs = causal_conv1d_forward(xc, w, activation="silu")
        y, state = selective_scan_forward(u.unflatten(-1, (H, P)), dt, A, B, C, D, bias)
        r, h = block_norm_forward(y.flatten(-2), gate=u, gate_first=True, post_weight=pre, pre_weight=pre)
        return u, cs, y, state, r, h

    want = [t.clone() for t in all_of_them()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_of_them()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = all_of_them()
    for seed in range(3):
        xc.copy_(_randn(_gen(seed), 2, n, c, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(all_of_them(), replayed)), seed


def test_timing_names_the_kernels():
    _lib.timing_reset()
    _lib.timing_enable(True)
    x = torch.randn(2, 8, 16, device=DEV)
    causal_conv1d_forward(x, torch.randn(16, 4, device=DEV))
    block_norm_forward(x, pre_weight=torch.ones(16, device=DEV))
    selective_scan_step(torch.zeros(2, 2, 8, 16, device=DEV), x[:, 0].unflatten(-1, (2, 8)), x[:, 0, :2], -torch.ones(2, device=DEV),
                        x[:, :1], x[:, 1:2])
    torch.cuda.synchronize()
    stats = _lib.timing_collect()
    _lib.timing_enable(False)
    assert {"causal_conv1d", "block_norm", "scan_seq"} <= {k for k, (c, _) in stats.items() if c}
