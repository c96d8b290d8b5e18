"""The state space operators without a GPU: the host forms against the 64-bit
oracle, the refusals of the entry points and of the C ABI."""

import ctypes

import pytest
import torch

from oracle import state_space as ora
from sparseflow_amd import _lib
from sparseflow_amd.Kernels.block_norm import block_norm_forward
from sparseflow_amd.Kernels.causal_conv1d import causal_conv1d_forward, causal_conv1d_step
from sparseflow_amd.Kernels.selective_scan import selective_scan_forward, selective_scan_step


def _scan_case(n=9, H=4, P=6, G=2, N=5, batch=2, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    return dict(x=r(batch, n, H, P), dt=r(batch, n, H), A=-torch.rand(H, generator=g) * 4, B=r(batch, n, G, N),
                C=r(batch, n, G, N), D=r(H), dt_bias=r(H))


def test_host_scan_prompt_packed_and_steps_agree_with_the_oracle():
    k = _scan_case()
    y, state = selective_scan_forward(**k)
    for b in range(2):
        ref, h, _, _ = ora.scan(k["x"][b], k["dt"][b], k["A"], k["B"][b], k["C"][b], k["D"], k["dt_bias"], True,
                                torch.zeros(4, 6, 5))
        assert torch.allclose(y[b].double(), ref, atol=1e-5) and torch.allclose(state[b].double(), h, atol=1e-5)
    flat = {n: (t.flatten(0, 1) if n in ("x", "dt", "B", "C") else t) for n, t in k.items()}
    off = torch.tensor([0, 9, 9, 18], dtype=torch.int32)
    yp, sp = selective_scan_forward(**flat, offsets=off)
    assert torch.equal(yp, y.flatten(0, 1)) and torch.equal(sp[[0, 2]], state) and not sp[1].any()
    pool = torch.zeros(5, 4, 6, 5)
    slots = torch.tensor([3, 0], dtype=torch.int32)
    for t in range(9):
        yt = selective_scan_step(pool, k["x"][:, t], k["dt"][:, t], k["A"], k["B"][:, t], k["C"][:, t], k["D"],
                                 k["dt_bias"], slots=slots)
        assert torch.equal(yt, y[:, t])
    assert torch.equal(pool[[3, 0]], state)
    yt = selective_scan_step(pool, k["x"][:, 0], k["dt"][:, 0], k["A"], k["B"][:, 0], k["C"][:, 0],
                             slots=torch.tensor([-1, 5], dtype=torch.int32))
    assert not yt.any() and torch.equal(pool[[3, 0]], state)


def test_host_conv_prompt_packed_and_steps_agree_with_the_oracle():
    g = torch.Generator().manual_seed(1)
    x, w, b = torch.randn(2, 7, 5, generator=g), torch.randn(5, 4, generator=g), torch.randn(5, generator=g)
    before = torch.randn(2, 3, 5, generator=g)
    y, state = causal_conv1d_forward(x, w, b, activation="silu", initial_state=before)
    for i in range(2):
        ref, last, _ = ora.conv1d(x[i], w, b, "silu", before[i])
        assert torch.allclose(y[i].double(), ref, atol=1e-5) and torch.equal(state[i].double(), last)
    yp, sp = causal_conv1d_forward(x.flatten(0, 1), w, b, activation="silu", initial_state=before,
                                   offsets=torch.tensor([0, 7, 14], dtype=torch.int32))
    assert torch.equal(yp, y.flatten(0, 1)) and torch.equal(sp, state)
    pool = before.clone()
    for t in range(7):
        assert torch.allclose(causal_conv1d_step(pool, x[:, t], w, b, activation="silu"), y[:, t], atol=1e-6)
    assert torch.equal(pool, state)


def test_host_block_norm_agrees_with_the_oracle():
    g = torch.Generator().manual_seed(2)
    x, gate, res = (torch.randn(3, 4, 24, generator=g) for _ in range(3))
    post, pre, scale = (torch.rand(24, generator=g) for _ in range(3))
    r, h = block_norm_forward(x, gate=gate[:, :1], gate_first=True, post_weight=post, group_size=8, residual=res,
                              scale=scale, pre_weight=pre, eps=1e-5)
    rr, hh, _ = ora.block_norm(x, gate[:, :1], "silu", True, post, 8, res, scale, pre, 1e-5)
    assert torch.allclose(r.double(), rr, atol=1e-5) and torch.allclose(h.double(), hh, atol=1e-5)


def test_scan_refusals():
    k = _scan_case()

    def bad(error=ValueError, **change):
        with pytest.raises(error):
            selective_scan_forward(**{**k, **change})

    bad(x=k["x"][0])
    bad(dt=k["dt"][:, :, :2])
    bad(dt=k["dt"].half())
    bad(B=k["B"][:, :-1])
    bad(C=k["C"][..., :-1])
    bad(B=torch.randn(2, 9, 3, 5), C=torch.randn(2, 9, 3, 5))  # 3 groups of 4 heads
    bad(A=k["A"].double())
    bad(A=None)
    bad(D=k["D"][:2])
    bad(dt_bias=torch.randn(8)[::2])
    bad(initial_state=torch.zeros(3, 4, 6, 5))
    bad(initial_state=torch.zeros(2, 4, 6, 5, dtype=torch.half))
    bad(final_state=torch.zeros(2, 4, 5, 6).transpose(2, 3))
    bad(slots=torch.zeros(2, dtype=torch.int32))  # no pool
    bad(slots=torch.zeros(2), final_state=torch.zeros(4, 4, 6, 5))
    bad(out=torch.zeros(2, 9, 4, 7))
    bad(_lib.UnsupportedError, x=k["x"].double(), dt=k["dt"].double(), B=k["B"].double(), C=k["C"].double())
    bad(_lib.UnsupportedError, B=torch.zeros(2, 9, 2, 257), C=torch.zeros(2, 9, 2, 257))
    flat = {n: (t.flatten(0, 1) if n in ("x", "dt", "B", "C") else t) for n, t in k.items()}
    for off in (torch.zeros(0, dtype=torch.int32), torch.tensor([0, 18]), torch.zeros(2, 2, dtype=torch.int32)):
        with pytest.raises(ValueError):
            selective_scan_forward(**flat, offsets=off)
    with pytest.raises(ValueError):
        selective_scan_step(torch.zeros(3, 4, 6, 5), k["x"][:, 0], k["dt"][:, 0], k["A"], k["B"][:, 0], k["C"][:, 0])


def test_conv_and_norm_refusals():
    x, w = torch.randn(2, 7, 5), torch.randn(5, 4)
    for kw in (dict(weight=torch.randn(6, 4)), dict(weight=w.half()), dict(weight=w[:, 0]), dict(bias=torch.randn(4)),
               dict(activation="relu"), dict(initial_state=torch.zeros(2, 4, 5)), dict(x=x[0]),
               dict(out=torch.zeros(2, 7, 6)), dict(slots=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            causal_conv1d_forward(**{**dict(x=x, weight=w), **kw})
    with pytest.raises(_lib.UnsupportedError):
        causal_conv1d_forward(x, torch.randn(5, 9))
    with pytest.raises(_lib.UnsupportedError):
        causal_conv1d_forward(x.double(), w)
    with pytest.raises(ValueError):
        causal_conv1d_step(torch.zeros(2, 3, 5), x, w)
    r = torch.randn(4, 24)
    for kw in (dict(group_size=7), dict(activation="tanh"), dict(pre_weight=torch.ones(23)), dict(gate=r.half()),
               dict(residual=r.half()), dict(scale=torch.ones(3)), dict(post_weight=torch.ones(24).double()),
               dict(out=torch.zeros(4, 24)), dict(residual_out=torch.zeros(4, 25)),
               dict(out=torch.zeros(4, 24).half(), pre_weight=torch.ones(24))):
        with pytest.raises(ValueError):
            block_norm_forward(r, **kw)
    with pytest.raises(_lib.UnsupportedError):
        block_norm_forward(torch.zeros(1, 16385))
    with pytest.raises(_lib.UnsupportedError):
        block_norm_forward(r.double())


def test_the_c_abi_refuses_before_it_touches_the_device():
    L, p = _lib.lib(), ctypes.c_void_p(64)
    INV, UNS = _lib.SF_ERR_INVALID, _lib.SF_ERR_UNSUPPORTED
    conv = lambda **k: _lib.Conv1dDesc(**{**dict(batch=1, tokens=4, max_len=4, states=1, x_strides=(32, 8), y_strides=(32, 8), channels=8, kernel=4), **k})  # noqa: E731,E501
    call = lambda d: L.sf_causal_conv1d(ctypes.byref(d), p, p, None, None, None, None, p, None, None)  # noqa: E731
    assert call(conv(kernel=9)) == UNS and call(conv(channels=0)) == INV and call(conv(batch=-1)) == INV
    assert call(conv(activation=2)) == UNS and call(conv(dtype=5)) == INV
    assert L.sf_causal_conv1d(None, p, p, None, None, None, None, p, None, None) == INV
    assert L.sf_causal_conv1d(ctypes.byref(conv()), None, p, None, None, None, None, p, None, None) == INV
    assert call(conv(batch=0)) == _lib.SF_OK
    scan = lambda **k: _lib.ScanDesc(**{**dict(batch=1, tokens=4, max_len=4, states=1, heads=4, head_dim=8, groups=2, state_dim=16), **k})  # noqa: E731,E501
    run = lambda d: L.sf_selective_scan(ctypes.byref(d), p, p, p, p, p, None, None, None, None, None, p, None, None, 0, None)  # noqa: E731,E501
    assert run(scan(groups=3)) == INV and run(scan(state_dim=257)) == UNS and run(scan(head_dim=0)) == INV
    assert run(scan(dtype=9)) == INV and run(scan(tokens=-1)) == INV and run(scan(batch=0)) == _lib.SF_OK
    assert run(scan(batch=1 << 31)) == UNS
    step = lambda d, s: L.sf_selective_scan_step(ctypes.byref(d), s, p, p, p, p, p, None, None, None, p, None)  # noqa: E731,E501
    assert step(scan(), None) == INV and step(scan(states=-1), p) == INV
    norm = lambda **k: _lib.NormDesc(**{**dict(outer=1, inner=2, dim=8, group_size=8), **k})  # noqa: E731
    do = lambda d, pre=None, r=p, h=None: L.sf_block_norm(ctypes.byref(d), p, None, None, None, None, pre, r, h, None)  # noqa: E731,E501
    assert do(norm(group_size=3)) == INV and do(norm(dim=16385, group_size=16385)) == UNS
    assert do(norm(residual_dtype=_lib.SF_F16)) == UNS and do(norm(activation=3)) == UNS
    assert do(norm(), r=None) == INV and do(norm(), pre=p) == INV and do(norm(), h=p) == INV
    assert do(norm(outer=0)) == _lib.SF_OK
