"""Checks of the modules over the 4-bit operators, for a device or the host."""

import copy

import torch
import torch.nn as nn

from oracle import mx4 as ora
from sparseflow_amd.Kernels.mx4 import mx4_quantize
from sparseflow_amd.Models import spiking_ssm_hybrid_tiny
from sparseflow_amd.neuron import reset_net
from sparseflow_amd.Ops import CachedAttention, MX4Linear, SparseLinear
from tests.mx4_checks import PARTS, STEP, attention_bound, half_step, within


def check_linear_module(dev, dtype, bias, quantize_input, sparse=False):
    torch.manual_seed(1)
    lin = nn.Linear(70, 36, bias=bias)
    lin = (SparseLinear.from_dense(lin) if sparse else lin).to(dev)
    mod = MX4Linear.from_dense(lin, quantize_input).to(dtype)
    x = torch.randn(3, 5, 70, generator=torch.Generator().manual_seed(2)).to(dtype).to(dev)
    y = mod(x)
    assert y.shape == (3, 5, 36) and y.dtype == dtype
    wv = ora.values(*mx4_quantize(lin.weight.detach()), 70)
    xv = ora.values(*mx4_quantize(x), 70) if quantize_input else x
    b = None if not bias else lin.bias.detach().to(dtype)
    ref, mag = ora.linear(xv.reshape(15, 70), wv, b)
    within(y.reshape(15, 36), ref, (PARTS[dtype] * 70 + 4) * STEP * mag + half_step(dtype) * ref.abs())
    assert torch.equal(mod.dequantized_weight().cpu().double(), wv)
    other = MX4Linear(70, 36, bias, quantize_input, dev).to(dtype)
    other.load_state_dict(mod.state_dict())
    assert torch.equal(other(x), y)


def _sequences(dev, batch, tokens, heads, kv, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(batch, tokens, h, dim, generator=g).to(dtype).to(dev) for h in (heads, kv, kv)]


def check_cached_attention(dev, dtype, page, parts, heads=4, kv=2, dim=33, batch=3):
    """Parts of any lengths, one after another, are the whole; against the oracle."""
    tokens = sum(parts)
    q, k, v = _sequences(dev, batch, tokens, heads, kv, dim, dtype)
    mod = CachedAttention(page_size=page)
    ys, at = [], 0
    for n in parts:
        ys.append(mod(*(t[:, at:at + n] for t in (q, k, v))))
        at += n
    y = torch.cat(ys, 1)
    held = [ora.values(*mx4_quantize(t.contiguous()), dim) for t in (k, v)]
    see = torch.arange(tokens)[None] <= torch.arange(tokens)[:, None]
    for b in range(batch):
        for h in range(heads):
            ref, mag, big = ora.attend(q[b, :, h], *(t[b, :, h // (heads // kv)] for t in held), see, dim ** -0.5)
            within(y[b, :, h], ref, attention_bound(dtype, dim, tokens, ref, mag, big), f"{b} {h}")
    assert int((mod.state.refs > 0).sum()) == batch * -(-tokens // page)


def check_select(dev, page, before, after):
    """The sequences of a search: those that go on have what their parents had, to the bit."""
    batch, steps = 4, [[2, 0, 2, 1], [3, 3, 3, 3], [0, 1, 2, 3]]
    total = before + after * len(steps)
    q, k, v = _sequences(dev, batch, total, 4, 1, 64, torch.float32, seed=3)
    part = lambda at, n: [t[:, at:at + n] for t in (q, k, v)]  # noqa: E731
    mod = CachedAttention(page_size=page)
    mod(*part(0, before))
    at = before
    line = [t[:, :before] for t in (q, k, v)]  # what each sequence is made of
    for i, p in enumerate(steps):
        p = torch.tensor(p)
        mod.select(p.to(dev) if i % 2 else p)
        if i == 1:
            mod.compact()
            assert mod.state.refs.numel() == int((mod.state.refs > 0).sum())
        y = mod(*part(at, after))
        line = [torch.cat([t[p.to(dev)], n], 1) for t, n in zip(line, part(at, after))]
        at += after
        alone = CachedAttention(page_size=page)
        alone(*(t[:, :-after] for t in line))
        assert torch.equal(y, alone(*(t[:, -after:] for t in line)))
    s = mod.state
    rows = s.tables[s.slots.long()][:, :-(-total // page)]
    count = torch.bincount(rows.flatten().long().cpu(), minlength=s.refs.numel())
    assert torch.equal(count, s.refs.cpu().long())  # every page is as often in use as the tables say


def hybrid(seed=0, vocab=32):
    torch.manual_seed(seed)
    m = spiking_ssm_hybrid_tiny(vocab=vocab, v_threshold=0.5).eval()
    with torch.no_grad():
        for mod in m.modules():
            if isinstance(mod, nn.Linear):
                mod.weight.copy_(mod.weight.to(torch.bfloat16).float())
    return m


def ids(batch, tokens, vocab=32, seed=1):
    return torch.randint(0, vocab, (batch, tokens), generator=torch.Generator().manual_seed(seed))


def search(model, dev, prompt, steps):
    """A beam search's calls with given parents and tokens -> all logits."""
    reset_net(model)
    with torch.no_grad():
        out = [model(prompt.to(dev))]
        for parents, token in steps:
            model.select(torch.tensor(parents))
            out.append(model(token.to(dev)))
    return torch.cat(out, 1).cpu()


def dequantized(model):
    """The same model with float weights that are what quantize_() would keep."""
    m = copy.deepcopy(model)
    with torch.no_grad():
        for mod in m.modules():
            if isinstance(mod, nn.Linear):
                mod.weight.copy_(ora.values(*mx4_quantize(mod.weight), mod.weight.shape[1]).float())
    return m
