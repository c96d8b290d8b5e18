"""The causal convolution and the block norm on the GPU at their edges, against the
64-bit oracle."""

import pytest
import torch

from oracle import state_space as ora
from sparseflow_amd.Kernels.block_norm import block_norm_forward
from sparseflow_amd.Kernels.causal_conv1d import causal_conv1d_forward, causal_conv1d_step
from sparseflow_amd.Kernels.selective_scan import selective_scan_forward
from sparseflow_amd.Models import spiking_ssm_tiny
from tests.gpu_helpers import DEV, announce

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _gates(dtype=F32):
    v = torch.cat([torch.linspace(-87, 20, 4091), torch.tensor([0.0, -0.0, 1e-8, -1e-8, 60.0])])
    return v.to(dtype)


def _close_to_a_few_units(got, want, what):
    # The exponential and the reciprocal are good to 2 half units each, and the sum, the
    # product and the correction to one: 7, and 10 are allowed.
    got = got.detach().double().cpu()
    off = (got - want).abs() - (10 * 2.0 ** -24 * want.abs() + 2.0 ** -126)
    assert bool((off <= 0).all()), f"{what}: worst {float(((got - want).abs() / want.abs().clamp(min=1e-300)).max()) * 2 ** 24:.3g} half units"


def test_float32_silu_of_the_convolution_to_its_last_bits():
    announce("conv silu float32")
    v = _gates()
    x, w = v.expand(3, -1).contiguous()[None], torch.ones(v.numel(), 1)
    y, _ = causal_conv1d_forward(x.to(DEV), w.to(DEV), activation="silu")
    want = ora.silu(v.double()).expand(1, 3, -1)
    _close_to_a_few_units(y, want, "prompt")
    step = causal_conv1d_step(torch.empty(3, 0, v.numel(), device=DEV), x[0].to(DEV), w.to(DEV), activation="silu")
    _close_to_a_few_units(step, want[0], "step")
    out = causal_conv1d_forward(torch.tensor([[[float("-inf"), float("inf"), -1e30, 1e30]]], device=DEV),
                                torch.ones(4, 1, device=DEV), activation="silu")[0].flatten().tolist()
    assert out[0] != out[0] and out[1] == float("inf") and out[2] == 0 and out[3] == torch.tensor(1e30).item()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
def test_gates_of_float32_results_to_their_last_bits(dtype, act):
    announce(f"norm gate {act} {dtype} to float32")
    g = _gates(dtype)
    x, residual = torch.ones(2, g.numel(), dtype=dtype), torch.zeros(2, g.numel())
    r, _ = block_norm_forward(x.to(DEV), gate=g.expand(2, -1).contiguous().to(DEV), activation=act,
                              residual=residual.to(DEV))
    assert r.dtype == F32
    v = g.double()
    _close_to_a_few_units(r, (ora.silu(v) if act == "silu" else torch.sigmoid(v)).expand(2, -1), act)


def test_outputs_that_overlap_inputs_are_refused():
    announce("overlapping outputs")
    x, w = torch.randn(2, 90, 48, device=DEV), torch.randn(48, 4, device=DEV)
    with pytest.raises(ValueError, match="shares memory with x"):
        causal_conv1d_forward(x, w, out=x)
    B, dt, A = torch.randn(2, 90, 1, 8, device=DEV), torch.randn(2, 90, 3, device=DEV), -torch.ones(3, device=DEV)
    xs = x.unflatten(-1, (3, 16))
    with pytest.raises(ValueError, match="shares memory with x"):
        selective_scan_forward(xs, dt, A, B, B, out=xs)
    pool = torch.zeros(3, 3, 16, 8, device=DEV)
    with pytest.raises(ValueError, match="shares memory with initial_state"):
        selective_scan_forward(xs, dt, A, B, B, initial_state=pool[:2], final_state=pool[1:])
    with pytest.raises(ValueError, match="workspace"):
        selective_scan_forward(xs, dt, A, B, B, workspace=torch.zeros(1, device=DEV).expand(1 << 20))
    wide = torch.randn(2, 90, 96, device=DEV)
    want = causal_conv1d_forward(wide[..., :48].contiguous(), w)[0]
    got = causal_conv1d_forward(wide[..., :48], w, out=wide[..., 48:])[0]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("dim,group", [(64, 64), (2048, 256), (999, 999), (4096, 4096)])
def test_a_norms_outputs_may_be_its_inputs(dtype, dim, group):
    announce(f"norm in place {dtype} {dim}")
    g = torch.Generator().manual_seed(dim)
    x, gate, residual = (torch.randn(37, dim, generator=g).to(dtype).to(DEV) for _ in range(3))
    post, pre = (torch.rand(dim, generator=g).to(DEV) for _ in range(2))
    kw = dict(post_weight=post, group_size=group, pre_weight=pre)
    want = block_norm_forward(x, gate=gate, residual=residual, **kw)
    for out, residual_out in (("x", "residual"), ("residual", "x"), ("gate", "residual"), ("x", "gate")):
        t = {"x": x.clone(), "gate": gate.clone(), "residual": residual.clone()}
        got = block_norm_forward(t["x"], gate=t["gate"], residual=t["residual"], out=t[out], residual_out=t[residual_out], **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_model_in_16_bits(dtype):
    announce(f"spiking ssm in {dtype}")
    torch.manual_seed(4)
    m = spiking_ssm_tiny(vocab=32, v_threshold=0.5).eval().to(DEV).to(dtype)
    ids = torch.randint(0, 32, (2, 40), device=DEV)
    with torch.no_grad():
        b, x = m.blocks[0], torch.randn(2, 40, m.blocks[0].mixed, device=DEV).to(dtype)
        want, _ = causal_conv1d_forward(x, b.conv.weight.float(), b.conv.bias.float(), activation="silu")
        assert torch.equal(b.conv(x), want)
        b.conv.reset()
        logits, more = m(ids), m(ids[:, :1])
    assert logits.shape == (2, 40, 32) and more.shape == (2, 1, 32) and logits.dtype == dtype
    assert torch.isfinite(logits).all() and torch.isfinite(more).all()


@pytest.mark.parametrize("shape", [(2, 3, 0, 8), (0, 3, 5, 8), (2, 0, 5, 8), (1, 1, 0, 2, 8), (0, 8), (3, 0, 8)])
def test_norms_over_empty_axes(shape):
    announce(f"norm over empty axes {shape}")
    x, w = torch.randn(shape, device=DEV), torch.rand(8, device=DEV)
    for gate in (None, x, torch.randn(8, device=DEV)):
        r, h = block_norm_forward(x, gate=gate, residual=x, pre_weight=w)
        assert r.shape == h.shape == x.shape


def test_a_norms_inputs_broadcast_or_are_refused():
    announce("norm broadcasts")
    x, w = torch.randn(3, 8, device=DEV), torch.rand(8, device=DEV)
    for shape in ((3, 7), (2, 8), (2, 3, 8), (1, 3, 8), (0, 8), (5,)):
        for name in ("gate", "residual"):
            with pytest.raises(ValueError, match="broadcast"):
                block_norm_forward(x, pre_weight=w, **{name: torch.randn(shape, device=DEV)})
    for shape in ((3, 8), (1, 8), (3, 1), (8,), (1,), ()):
        t = torch.randn(shape, device=DEV)
        got = block_norm_forward(x, gate=t, residual=t, pre_weight=w)
        want = block_norm_forward(x, gate=t.expand(3, 8).contiguous(), residual=t.expand(3, 8).contiguous(), pre_weight=w)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
