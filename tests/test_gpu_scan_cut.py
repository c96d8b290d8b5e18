"""Scans whose token axis is cut into segments: states kept in place.

The same call with separate pools runs the same arithmetic, so that results are the
same bit for bit."""

import pytest
import torch

from oracle import state_space as ora
from sparseflow_amd import _lib
from sparseflow_amd.Kernels.selective_scan import selective_scan_forward
from sparseflow_amd.Ops import SelectiveScan
from tests.gpu_helpers import DEV, announce

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _inputs(lead, H, P, G, N, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    return ((r(*lead, H, P)).to(dtype).to(DEV), r(*lead, H).to(dtype).to(DEV), (-torch.rand(H, generator=g) - 0.1).to(DEV),
            (r(*lead, G, N) / N ** 0.5).to(dtype).to(DEV), r(*lead, G, N).to(dtype).to(DEV))


def _kernels(run):
    _lib.timing_reset()
    _lib.timing_enable(True)
    out = run()
    torch.cuda.synchronize()
    stats = _lib.timing_collect()
    _lib.timing_enable(False)
    return out, {k for k, (c, _) in stats.items() if c}


def _both_ways(args, pool, **kw):
    apart = pool.clone()
    want, names = _kernels(lambda: selective_scan_forward(*args, initial_state=pool, final_state=apart, **kw))
    assert "scan_parts" in names, "the call is not cut"
    start = pool.clone()
    y, kept = selective_scan_forward(*args, initial_state=pool, final_state=pool, **kw)
    assert kept is pool and torch.equal(y, want[0]) and torch.equal(pool, apart)
    return y, start


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch,n,H,P,G,N", [(1, 1111, 2, 32, 1, 32), (3, 700, 4, 40, 2, 70), (2, 4096, 24, 64, 1, 128)])
def test_dense_in_place(dtype, batch, n, H, P, G, N):
    announce(f"scan cut in place {dtype} {batch}x{n} H={H} P={P} N={N}")
    args = _inputs((batch, n), H, P, G, N, dtype, n)
    pool = torch.randn(batch, H, P, N, generator=torch.Generator().manual_seed(1)).to(DEV)
    y, start = _both_ways(args, pool)
    if n < 1200:
        x, dt, A, B, C = (t.cpu() for t in args)
        for b in range(batch):
            ref, h, ym, hm = ora.scan(x[b], dt[b], A, B[b], C[b], None, None, True, start[b].cpu())
            f = (4 * n + 300) * 2.0 ** -24
            assert bool(((pool[b].double().cpu() - h).abs() <= f * hm).all())
            half_ulp, inner = {F32: (2.0 ** -24, 0), F16: (2.0 ** -11, 2.0 ** -15), BF16: (2.0 ** -8, 2.0 ** -8)}[dtype]
            assert bool(((y[b].double().cpu() - ref).abs() <= (f + inner) * ym + half_ulp * ref.abs() + 2.0 ** -25).all())


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("longest,others,H,N", [(8192, 63, 24, 128), (3000, 20, 8, 64), (2049, 7, 4, 48)])
def test_packed_in_place_with_more_workgroups_than_places(dtype, longest, others, H, N):
    """One long sequence sets the segments, and sequences that end just inside one of
    them have a last segment that is done long before the others."""
    announce(f"scan cut in place packed {dtype} {longest} + {others} H={H} N={N}")
    g = torch.Generator().manual_seed(longest)
    lens = [longest] + [int(v) for v in torch.randint(1, 1000, (others,), generator=g)] + [0, 1]
    off = [0]
    for v in lens:
        off.append(off[-1] + v)
    args = _inputs((off[-1],), H, 64, 1, N, dtype, others)
    rows = len(lens) + 4
    pool = torch.randn(rows, H, 64, N, generator=g).to(DEV)
    slots = torch.randperm(rows, generator=g)[:len(lens)].to(torch.int32)
    slots[3] = -1  # starts from zeros and is not kept
    y, start = _both_ways(args, pool, slots=slots.to(DEV), offsets=torch.tensor(off, dtype=torch.int32, device=DEV),
                          max_len=longest)
    rest = [r for r in range(rows) if r not in slots.tolist()]
    assert torch.equal(pool[rest], start[rest])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_module_continues_long_prompts(dtype):
    announce(f"scan module long prompts {dtype}")
    torch.manual_seed(0)
    m = SelectiveScan(4, 32, 64).to(DEV)
    n = 1500
    x, dt, _, B, C = _inputs((1, 3 * n), 4, 32, 1, 64, dtype, 5)
    with torch.no_grad():
        m(x[:, :7], dt[:, :7], B[:, :7], C[:, :7])
        ys, state = [], m.state.clone()
        for i in range(3):
            at = slice(i * n, (i + 1) * n)
            ys.append((m(x[:, at], dt[:, at], B[:, at], C[:, at]), at, state))
            state = m.state.clone()
        A = -torch.exp(m.A_log)
        for y, at, before in ys:
            want, after = selective_scan_forward(x[:, at], dt[:, at], A, B[:, at], C[:, at], D=m.D, dt_bias=m.dt_bias,
                                                 initial_state=before)
            assert torch.equal(y, want)
        assert torch.equal(after, m.state)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens", [[5000] + [3, 0, 40, 1] * 40, [7, 3000, 0, 65, 129, 97, 33, 64, 2, 1025, 130, 131, 63] * 2,
                                  [100] * 30 + [2000], [4000] + [70] * 50])
def test_packed_long_among_short(dtype, lens):
    """The segments of cut sequences next to each other do not share workspace."""
    announce(f"scan packed long among short {dtype} {len(lens)} of up to {max(lens)}")
    H, P, G, N = 2, 32, 1, 16
    off = [0]
    for v in lens:
        off.append(off[-1] + v)
    args = _inputs((off[-1],), H, P, G, N, dtype, len(lens))
    pool = torch.randn(len(lens), H, P, N, generator=torch.Generator().manual_seed(2)).to(DEV)
    y, start = _both_ways(args, pool, offsets=torch.tensor(off, dtype=torch.int32, device=DEV), max_len=max(lens))
    x, dt, A, B, C = (t.cpu() for t in args)
    for i, n in enumerate(lens):
        at = slice(off[i], off[i + 1])
        ref, h, ym, hm = ora.scan(x[at], dt[at], A, B[at], C[at], None, None, True, start[i].cpu())
        f = (4 * n + 300) * 2.0 ** -24
        half_ulp, inner = {F32: (2.0 ** -24, 0), F16: (2.0 ** -11, 2.0 ** -15), BF16: (2.0 ** -8, 2.0 ** -8)}[dtype]
        assert bool(((pool[i].double().cpu() - h).abs() <= f * hm).all()), f"state {i} of {n}"
        assert bool(((y[at].double().cpu() - ref).abs() <= (f + inner) * ym + half_ulp * ref.abs() + 2.0 ** -25).all()), \
            f"sequence {i} of {n}"


@pytest.mark.parametrize("longest", [8, 200, 700])
def test_dense_calls_whose_longest_is_not_their_tokens(longest):
    """max_len only sizes the launch: of dense sequences too, where it should be their
    tokens."""
    announce(f"scan dense with max_len {longest}")
    n, H, P, G, N = 700, 3, 32, 1, 32
    x, dt, A, B, C = _inputs((2, n), H, P, G, N, F32, 9)
    want, last = selective_scan_forward(x, dt, A, B, C)
    y, state = torch.zeros_like(x), torch.zeros_like(last)
    desc = _lib.scan_desc(2, n, longest, 2, x.stride()[:3], dt.stride(), B.stride()[:3], C.stride()[:3], y.stride()[:3], H, P, G,
                          N, F32, True)
    workspace = torch.empty(max(desc[2], 16), dtype=torch.uint8, device=DEV)
    _lib.selective_scan(desc, x, dt, A, B, C, None, None, None, None, None, y, state, workspace)
    assert torch.allclose(y, want, rtol=1e-4, atol=1e-4) and torch.allclose(state, last, rtol=1e-4, atol=1e-4)
