"""The spiking state space model on the GPU: the optimized model (SparseLinear
projections, the state space kernels) against the host forms, prompts and tokens one
at a time.  Weights of the projections are bf16 values, so that the matrix-core
Linear's products are exact; of the ~15,000 neuron steps, each within ~1e-6 of the
host's membrane, about 0.02 are expected to lie that near their threshold, so the
spikes agree and the logits do to float32 rounding through four blocks."""

import copy

import pytest
import torch

import sparseflow_amd as sf
from sparseflow_amd import _lib
from sparseflow_amd.Models import spiking_ssm_tiny
from sparseflow_amd.neuron import reset_net
from sparseflow_amd.Ops import SparseLinear
from tests.gpu_helpers import DEV, announce, native_loaded

pytestmark = pytest.mark.gpu


def _model():
    torch.manual_seed(0)
    m = spiking_ssm_tiny(vocab=64, v_threshold=0.5).eval()
    with torch.no_grad():
        for mod in m.modules():
            if isinstance(mod, torch.nn.Linear):
                mod.weight.copy_(mod.weight.to(torch.bfloat16).float())
    return m


def test_prompt_then_tokens_match_the_host():
    announce("spiking ssm prompt and tokens")
    host = _model()
    dev = copy.deepcopy(host).to(DEV)
    ids = torch.randint(0, 64, (2, 40), generator=torch.Generator().manual_seed(1))
    sf.optimize(dev, sample_input=ids.to(DEV), verbose=False)
    assert sum(isinstance(m, SparseLinear) for m in dev.modules()) >= 8
    reset_net(dev)
    with torch.no_grad():
        want = host(ids)
        _lib.timing_reset()
        _lib.timing_enable(True)
        got = [dev(ids[:, :33].to(DEV))]
        for t in range(33, 40):
            got.append(dev(ids[:, t:t + 1].to(DEV)))
        torch.cuda.synchronize()
        stats = _lib.timing_collect()
        _lib.timing_enable(False)
    launched = {k for k, (c, _) in stats.items() if c}
    assert {"causal_conv1d", "scan_chunk", "scan_seq", "block_norm", "lif_multistep"} <= launched, launched
    got = torch.cat(got, 1).cpu()
    assert torch.isfinite(got).all()
    off = (got - want).abs().amax(-1)
    assert bool((off < 1e-3).all()), f"{int((off >= 1e-3).sum())} of {off.numel()} positions differ, most {float(off.max()):.3g}"
    assert native_loaded()


def test_bf16_prompts_of_a_block_run_the_direct_kernels():
    announce("spiking ssm block operators in bf16")
    m = _model().to(DEV).to(torch.bfloat16)
    b = m.blocks[0]
    for mod in (b.conv, b.scan, b.gate_norm):
        mod.float()  # (their parameters stay float32)
    g = torch.Generator().manual_seed(2)
    u = torch.randn(3, 70, b.mixed, generator=g).to(DEV, torch.bfloat16)
    dt = torch.randn(3, 70, b.heads, generator=g).to(DEV, torch.bfloat16)
    z = torch.randn(3, 70, b.inner, generator=g).to(DEV, torch.bfloat16)

    def run(u, dt, z):
        v = b.conv(u)
        x, B, C = v.split([b.inner, b.state_dim, b.state_dim], dim=-1)
        y = b.scan(x.unflatten(-1, (b.heads, b.head_dim)), dt, B[:, :, None], C[:, :, None])
        return b.gate_norm(y.flatten(-2), gate=z)[0]

    with torch.no_grad():
        whole = run(u, dt, z)
        reset_net(b)
        parts = [run(u[:, :50], dt[:, :50], z[:, :50])] + [run(u[:, t:t + 1], dt[:, t:t + 1], z[:, t:t + 1])
                                                         for t in range(50, 70)]
    # y is rounded to bf16 before the norm, once more in it, and its sums' operands are (2^-8 each).
    off = (torch.cat(parts, 1).float() - whole.float()).norm() / whole.float().norm()
    assert float(off) < 2.0 ** -7
