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
from sparseflow_amd.Kernels.selective_scan import selective_scan_forward
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
