"""Checks of the modules over the 4-bit operators, for a device or the host."""

import copy
import io

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


def check_select_of_nothing(dev):
    """Sequences without tokens, and a batch without sequences, go on like others."""
    q, k, v = _sequences(dev, 2, 3, 4, 2, 32, torch.float32)
    mod = CachedAttention(page_size=4)
    assert mod(q[:, :0], k[:, :0], v[:, :0]).shape == (2, 0, 4, 32)
    mod.select(torch.tensor([1, 1]))
    mod.compact()
    y = mod(q, k, v)
    assert torch.equal(y, CachedAttention(page_size=4)(q, k, v))
    mod = CachedAttention(page_size=4)
    assert mod(q[:0], k[:0], v[:0]).shape == (0, 3, 4, 32)
    mod.select(torch.zeros(0, dtype=torch.long))
    mod.compact()


def check_hybrid_in_16_bits(dev, dtype):
    """A prompt, its next token, and the sequences in other places, in a model of 16 bits."""
    m = hybrid(1).to(dev).to(dtype)
    with torch.no_grad():
        y = m(ids(2, 7).to(dev))
        m.select(torch.tensor([1, 1]))
        z = m(ids(1, 1).expand(2, 1).to(dev))
    assert y.dtype == dtype and y.shape == (2, 7, 32) and torch.isfinite(y).all()
    assert torch.equal(z[0], z[1]) and torch.isfinite(z).all()
    q = hybrid(1).quantize_().to(dev).to(dtype)
    with torch.no_grad():
        assert torch.isfinite(q(ids(2, 7).to(dev))).all()


def check_saved(dev):
    """A model in the middle of its sequences goes on after it was written and read, or copied."""
    m = hybrid(4).quantize_().to(dev)
    with torch.no_grad():
        m(ids(2, 5).to(dev))
        m.select(torch.tensor([1, 0]))
        file = io.BytesIO()
        torch.save(m, file)
        file.seek(0)
        others = [torch.load(file, weights_only=False), copy.deepcopy(m)]
        token = ids(2, 1, seed=8).to(dev)
        want = m(token)
        for other in others:
            assert torch.equal(other(token), want)
            other.select(torch.tensor([0, 0]))
            y = other(token[:1].expand(2, 1))  # (the same sequence twice, and the same next token)
            assert torch.equal(y[0], y[1])
