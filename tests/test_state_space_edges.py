"""The state space operators without a GPU: workspaces, arguments that must not be
taken for others, tensors that overlap, modules in 16 bits."""

import math
import pickle

import pytest
import torch

from sparseflow_amd import _lib
from sparseflow_amd.Kernels import block_norm
from sparseflow_amd.Kernels.block_norm import block_norm_forward
from sparseflow_amd.Kernels.causal_conv1d import causal_conv1d_forward, causal_conv1d_step
from sparseflow_amd.Kernels.selective_scan import selective_scan_forward, selective_scan_step
from sparseflow_amd.Models import spiking_ssm_tiny
from sparseflow_amd.Ops import BlockNorm, CausalConv1d, SelectiveScan


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("each", [1, 16])
def test_a_scans_workspace_is_of_the_sequences_that_are_cut(dtype, each):
    """One long sequence among short ones: no workspace times the whole batch."""
    H, P, N, long, short = 64, 64, 128, 16384, 255
    tokens = long + short * each
    desc = _lib.scan_desc(short + 1, tokens, long, short + 1, *[(0, 1, 1)] * 5, H, P, 1, N, dtype, True)
    data = tokens * 2 * H * P * dtype.itemsize + 2 * (short + 1) * H * P * N * 4
    assert 0 < desc[2] < data // 4, f"{desc[2]} bytes of workspace for {data} of data"


def _conv(n=6, c=4):
    return torch.randn(2, n, c), torch.randn(c, 3)


def _scan(n=5, H=2, P=4, G=1, N=3):
    return [torch.randn(2, n, H, P), torch.randn(2, n, H), -torch.rand(H), torch.randn(2, n, G, N), torch.randn(2, n, G, N)]


def test_a_convolutions_outputs_share_no_memory_with_its_inputs():
    x, w = _conv()
    buffer = torch.randn(2, 9, 4)
    pools = torch.zeros(3, 2, 4)
    flat = torch.zeros(40)
    for kw in (dict(x=x, out=x), dict(x=buffer[:, :6], out=buffer[:, 1:7]), dict(x=buffer[:, :6], out=buffer[:, 3:]),
               dict(x=x, initial_state=pools[:2], final_state=pools[1:]),
               dict(x=x, initial_state=flat[:16].view(2, 2, 4), final_state=flat[1:17].view(2, 2, 4)),
               dict(x=x, out=torch.zeros(1, 6, 4).expand(2, 6, 4))):
        with pytest.raises(ValueError, match="memory|expanded"):
            causal_conv1d_forward(**kw, weight=w)
    want, _ = causal_conv1d_forward(x, w)
    # Side by side in one buffer, along any axis, is apart.
    for place in (torch.zeros(2, 12, 4), torch.zeros(2, 6, 8), torch.zeros(4, 6, 4), torch.zeros(2, 6, 2, 4)):
        a, b = {(2, 12, 4): (place[:, :6], place[:, 6:]), (2, 6, 8): (place[..., :4], place[..., 4:]),
                (4, 6, 4): (place[:2], place[2:]), (2, 6, 2, 4): (place[:, :, 0], place[:, :, 1])}[tuple(place.shape)]
        for i, o in ((a, b), (b, a)):
            i.copy_(x)
            assert torch.equal(causal_conv1d_forward(i, w, out=o)[0], want) and torch.equal(i, x)
    state = torch.zeros(2, 2, 4)
    y, kept = causal_conv1d_forward(x, w, initial_state=state, final_state=state)
    assert kept is state and torch.equal(y, want)
    xt, s1, s2 = x[:, 0].clone(), state.clone(), state.clone()
    want = causal_conv1d_step(s1, xt, w)
    got = causal_conv1d_step(s2, xt, w, out=xt)
    assert got is xt and torch.equal(got, want) and torch.equal(s1, s2)
    with pytest.raises(ValueError, match="memory"):
        causal_conv1d_step(state, xt, w, out=state[:, 0])


def test_a_scans_outputs_share_no_memory_with_its_inputs():
    x, dt, A, B, C = _scan()
    buffer, states = torch.randn(2, 5, 2, 12), torch.zeros(3, 2, 4, 3)
    for kw in (dict(x=x, out=x), dict(x=buffer[..., :4], out=buffer[..., 3:7]),
               dict(x=x, initial_state=states[:2], final_state=states[1:]), dict(x=x, workspace=torch.zeros(1).expand(1 << 20)),
               dict(x=x, out=torch.zeros(1, 5, 2, 4).expand(2, 5, 2, 4))):
        with pytest.raises(ValueError, match="memory|expanded|contiguous"):
            selective_scan_forward(**{**dict(dt=dt, A=A, B=B, C=C), **kw})
    wide = torch.zeros(2, 5, 8)
    with pytest.raises(ValueError, match="shares memory with B"):
        selective_scan_forward(x, dt, A, wide[..., 2:5].unsqueeze(2), C, out=wide.unflatten(-1, (2, 4)))
    want, last = selective_scan_forward(x, dt, A, B, C)
    row = torch.zeros(2, 5, 8 + 8 + 6)
    xs, out = row[..., :8].unflatten(-1, (2, 4)), row[..., 8:16].unflatten(-1, (2, 4))
    Bs, Cs = row[..., 16:19].unsqueeze(2), row[..., 19:].unsqueeze(2)
    xs.copy_(x), Bs.copy_(B), Cs.copy_(C)
    assert torch.equal(selective_scan_forward(xs, dt, A, Bs, Cs, out=out)[0], want)
    assert torch.equal(xs, x) and torch.equal(Bs, B) and torch.equal(Cs, C)
    s1, s2, xt = torch.zeros(2, 2, 4, 3), torch.zeros(2, 2, 4, 3), x[:, 0].clone()
    want = selective_scan_step(s1, xt, dt[:, 0], A, B[:, 0], C[:, 0])
    assert torch.equal(selective_scan_step(s2, xt, dt[:, 0], A, B[:, 0], C[:, 0], out=xt), want) and torch.equal(s1, s2)
    with pytest.raises(ValueError, match="memory"):
        selective_scan_step(s1, x[:, 0], dt[:, 0], A, B[:, 0], C[:, 0], out=s1.view(-1)[:16].view(2, 2, 4))


def test_a_norms_outputs_are_its_inputs_or_apart():
    x, residual, w = torch.randn(3, 5, 8), torch.randn(3, 5, 8), torch.rand(8)
    want_r, want_h = block_norm_forward(x, gate=x, residual=residual, pre_weight=w)
    for out, residual_out in (("x", "residual"), ("residual", "x"), (None, "x"), ("x", None)):
        t = {"x": x.clone(), "residual": residual.clone(), None: None}
        r, h = block_norm_forward(t["x"], gate=t["x"], residual=t["residual"], pre_weight=w, out=t[out],
                                  residual_out=t[residual_out])
        assert torch.equal(r, want_r) and torch.equal(h, want_h)
    one = x[:1].clone()  # (strides of an axis of one do not matter)
    r, h = block_norm_forward(one, pre_weight=w, out=one.as_strided((1, 5, 8), (7, 8, 1)))
    assert torch.equal(one, block_norm_forward(x[:1], pre_weight=w)[1])
    buffer = torch.randn(4, 5, 8)
    row = torch.randn(5, 8)
    for kw in (dict(x=buffer[:3], out=buffer[1:]), dict(x=buffer[:3], residual_out=buffer[1:]),
               dict(x=x, gate=row.expand(3, 5, 8), out=row.expand(3, 5, 8)),
               dict(x=x, out=buffer[:3], residual_out=buffer[:3]), dict(x=x, out=buffer[:3], residual_out=buffer[1:])):
        with pytest.raises(ValueError, match="memory|expanded"):
            block_norm_forward(**kw, pre_weight=w)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_modules_in_16_bits(dtype):
    torch.manual_seed(3)
    conv, scan = CausalConv1d(8).to(dtype), SelectiveScan(2, 4, 3).to(dtype)
    norm = BlockNorm(8, post=True, pre=True, scale=0.5).to(dtype)
    x = torch.randn(2, 5, 8).to(dtype)
    dt, B = torch.randn(2, 5, 2).to(dtype), torch.randn(2, 5, 1, 3).to(dtype)
    for _ in range(2):
        y = conv(x)
        assert torch.equal(y, causal_conv1d_forward(x, conv.weight.float(), conv.bias.float(), activation="silu")[0])
        y = scan(x.unflatten(-1, (2, 4)), dt, B, B)
        want, _ = selective_scan_forward(x.unflatten(-1, (2, 4)), dt, -torch.exp(scan.A_log.float()), B, B, D=scan.D.float(),
                                         dt_bias=scan.dt_bias.float())
        assert y.dtype == dtype and torch.equal(y, want)
        r, h = norm(x, residual=x)
        want = block_norm_forward(x, post_weight=norm.post_weight.float(), residual=x, scale=norm.scale.float(),
                                  pre_weight=norm.pre_weight.float(), eps=norm.eps)
        assert torch.equal(r, want[0]) and torch.equal(h, want[1])
        # (A token after the prompt, and weights that have changed.)
        assert conv(x[:, :1]).shape == (2, 1, 8) and scan(x[:, :1].unflatten(-1, (2, 4)), dt[:, :1], B[:, :1], B[:, :1]).dtype == dtype
        conv.reset(), scan.reset()
        with torch.no_grad():
            for p in (*conv.parameters(), *scan.parameters(), *norm.parameters()):
                p.add_(0.5)


def test_a_model_in_16_bits():
    torch.manual_seed(4)
    m = spiking_ssm_tiny(vocab=32, v_threshold=0.5).eval().to(torch.bfloat16)
    ids = torch.randint(0, 32, (2, 6))
    with torch.no_grad():
        logits = m(ids)
        more = m(ids[:, :1])
    assert logits.shape == (2, 6, 32) and more.shape == (2, 1, 32) and torch.isfinite(logits).all()


def test_numbers_that_come_as_tensors_are_read_at_every_call():
    x, w = torch.randn(3, 8), torch.rand(8)
    eps, group, first = torch.tensor(1e-5), torch.tensor(8), torch.tensor(True)
    block_norm_forward(x, post_weight=w, eps=eps, group_size=group, gate=x, gate_first=first)
    eps.fill_(1.0), group.fill_(4), first.fill_(False)
    got, _ = block_norm_forward(x, post_weight=w, eps=eps, group_size=group, gate=x, gate_first=first)
    assert torch.equal(got, block_norm_forward(x, post_weight=w, eps=1.0, group_size=4, gate=x)[0])
    xs, dt, A, B, C = _scan()
    flat, off, longest, soft = [t.flatten(0, 1) for t in (xs, dt, B, C)], torch.tensor([0, 4, 10], dtype=torch.int32), \
        torch.tensor(6), torch.tensor(True)
    run = lambda most, plus: selective_scan_forward(flat[0], flat[1], A, *flat[2:], dt_softplus=plus, offsets=off, max_len=most)[0]  # noqa: E731
    assert torch.equal(run(longest, soft), run(6, True))
    longest.fill_(5), soft.fill_(False)
    assert torch.equal(run(longest, soft), run(5, False))


def test_a_norm_alone_returns_r_apart_from_x():
    x, w = torch.randn(3, 8), torch.rand(8)
    before = x.clone()
    r, _ = block_norm_forward(x, pre_weight=w)
    assert torch.equal(r, x)
    r.zero_()
    assert torch.equal(x, before)


@pytest.mark.parametrize("shape", [(2, 3, 0, 4), (0, 3, 5, 4), (2, 0, 5, 4), (2, 3, 5, 4), (1, 1, 0, 2, 4)])
def test_a_norms_rows_over_empty_axes(shape):
    """More than three axes become three, also where one of them is empty."""
    t = torch.randn(shape)
    rows, = block_norm._rows(t, t.shape)
    assert rows.shape == (math.prod(shape[:-2]), *shape[-2:])
    spread, = block_norm._rows(torch.randn(shape[-1]), t.shape)
    assert spread.shape == rows.shape


def test_a_norms_gate_and_residual_that_do_not_broadcast_are_refused():
    x, w = torch.randn(3, 8), torch.rand(8)
    for shape in ((3, 7), (2, 8), (2, 3, 8), (1, 3, 8), (0, 8), (5,)):
        for name in ("gate", "residual"):
            with pytest.raises(ValueError, match="broadcast"):
                block_norm_forward(x, pre_weight=w, **{name: torch.randn(shape)})
    for shape in ((3, 8), (1, 8), (3, 1), (8,), (1,), ()):
        t = torch.randn(shape)
        got = block_norm_forward(x, gate=t, residual=t, pre_weight=w)
        want = block_norm_forward(x, gate=t.expand(3, 8).contiguous(), residual=t.expand(3, 8).contiguous(), pre_weight=w)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_modules_are_pickled(dtype):
    torch.manual_seed(5)
    x, dt, B = torch.randn(2, 5, 8).to(dtype), torch.randn(2, 5, 2).to(dtype), torch.randn(2, 5, 1, 3).to(dtype)
    for m, args in ((CausalConv1d(8).to(dtype), (x,)), (SelectiveScan(2, 4, 3).to(dtype), (x.unflatten(-1, (2, 4)), dt, B, B)),
                    (BlockNorm(8, post=True).to(dtype), (x,)), (spiking_ssm_tiny(vocab=16).to(dtype), (torch.zeros(1, 3, dtype=torch.long),))):
        for used in (False, True):
            again = pickle.loads(pickle.dumps(m))
            for mod in (*m.modules(), *again.modules()):
                if hasattr(mod, "reset"):
                    mod.reset()
            with torch.no_grad():
                got, want = again(*args), m(*args)
            got, want = (t[0] if isinstance(t, tuple) else t for t in (got, want))
            assert torch.equal(got, want)
