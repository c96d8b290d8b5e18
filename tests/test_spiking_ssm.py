"""The spiking state space model on the CPU (host forms): prompts and tokens one at
a time give the same logits, states are the modules' own, optimize() replaces the
projections that spikes feed."""

import torch

import sparseflow_amd as sf
from sparseflow_amd.Models import spiking_ssm_tiny
from sparseflow_amd.neuron import reset_net
from sparseflow_amd.Ops import CausalConv1d, SelectiveScan, SparseLinear


def _model(seed=0):
    torch.manual_seed(seed)
    return spiking_ssm_tiny(vocab=32, v_threshold=0.5).eval()


def test_prompt_equals_its_tokens_one_by_one():
    m = _model()
    ids = torch.randint(0, 32, (2, 9), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        whole = m(ids)
        reset_net(m)
        parts = [m(ids[:, :5])] + [m(ids[:, t:t + 1]) for t in range(5, 9)]
    assert whole.shape == (2, 9, 32) and torch.isfinite(whole).all()
    assert torch.allclose(torch.cat(parts, 1), whole, atol=1e-4)
    states = [mod.state for mod in m.modules() if isinstance(mod, (CausalConv1d, SelectiveScan))]
    assert len(states) == 8 and all(s is not None for s in states)
    reset_net(m)
    assert all(mod.state is None for mod in m.modules() if isinstance(mod, (CausalConv1d, SelectiveScan)))


def test_sequences_of_a_batch_do_not_meet():
    m = _model(2)
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 32, (3, 6), generator=g)
    with torch.no_grad():
        both = m(ids)
        reset_net(m)
        alone = m(ids[1:2])
    assert torch.allclose(both[1:2], alone, atol=1e-5)


def test_optimize_replaces_the_projections():
    m = _model(4)
    ids = torch.randint(0, 32, (2, 4), generator=torch.Generator().manual_seed(5))
    with torch.no_grad():
        want = m(ids)
        reset_net(m)
        sf.optimize(m, sample_input=ids, verbose=False)
        reset_net(m)
        got = m(ids)
    for b in m.blocks:
        assert isinstance(b.in_proj, SparseLinear) and isinstance(b.out_proj, SparseLinear)
    assert torch.allclose(got, want, atol=1e-5)
