"""Modules over the 4-bit operators and the model that runs them, on the CPU (host forms)."""

import copy

import pytest
import torch
import torch.nn as nn

import sparseflow_amd as sf
from sparseflow_amd import _lib
from sparseflow_amd.Models import spiking_ssm_tiny
from sparseflow_amd.neuron import reset_net
from sparseflow_amd.Ops import CachedAttention, MX4Linear, quantize_linears_
from tests.mx4_module_checks import check_cached_attention, check_hybrid_in_16_bits, check_linear_module, \
    check_saved, check_select, check_select_of_nothing, dequantized, hybrid, ids, search

CPU = torch.device("cpu")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias,quantize_input,sparse", [(True, False, False), (False, True, False), (True, True, True)])
def test_linear_module(dtype, bias, quantize_input, sparse):
    check_linear_module(CPU, dtype, bias, quantize_input, sparse)


def test_quantize_linears_replaces_what_it_is_asked_for():
    shared = nn.Linear(32, 32)
    net = nn.ModuleDict({"a": shared, "b": shared, "c": nn.Linear(32, 8), "d": nn.Sequential(nn.Linear(8, 4), nn.ReLU())})
    assert quantize_linears_(net, only=lambda name, m: name != "c") == 3
    assert net["a"] is net["b"] and isinstance(net["a"], MX4Linear)
    assert isinstance(net["c"], nn.Linear) and isinstance(net["d"][0], MX4Linear)
    with pytest.raises(ValueError):
        net["a"](torch.zeros(2, 31))


@pytest.mark.parametrize("page,parts", [(1, [3, 1, 2]), (4, [7, 1, 1, 5, 1]), (64, [1, 1, 70])])
def test_cached_attention_module(page, parts):
    check_cached_attention(CPU, torch.float32, page, parts)


@pytest.mark.parametrize("page,before,after", [(4, 8, 1), (4, 6, 3), (1, 2, 1), (16, 5, 12)])
def test_select(page, before, after):
    check_select(CPU, page, before, after)


def test_cached_attention_refusals_leave_the_sequences():
    mod = CachedAttention(page_size=4)
    k = torch.randn(2, 3, 2, 8)
    q = torch.randn(2, 3, 4, 8)
    mod(q, k, k)
    for args, error in (((q, k.half(), k), ValueError), ((q, k, k[:, :2]), ValueError), ((q[:, :, :3], k, k), ValueError),
                        ((q[:, :2], k, k), ValueError), ((q.double(), k.double(), k.double()), _lib.UnsupportedError),
                        ((q[0], k, k), ValueError),
                        ((torch.zeros(2, 1, 1, 257),) + (torch.zeros(2, 1, 1, 257),) * 2, _lib.UnsupportedError)):
        with pytest.raises(error):
            mod(*args)
        assert mod.state.tokens == 3
    for parents in (torch.tensor([0, 2]), torch.tensor([-1, 0]), torch.tensor([0]), torch.tensor([0.0, 1.0])):
        with pytest.raises(ValueError):
            mod.select(parents)
    assert mod(q[:, :0], k[:, :0], k[:, :0]).shape == (2, 0, 4, 8) and mod.state.tokens == 3
    for page in (0, 3, 8192):
        with pytest.raises(ValueError):
            CachedAttention(page_size=page)
    assert mod(q[:1], k[:1], k[:1]).shape == (1, 3, 4, 8) and mod.state.tokens == 3  # (another batch begins anew)
    mod.reset()
    mod.select(torch.tensor([0]))
    mod.compact()


def test_hybrid_prompt_equals_its_tokens_one_by_one():
    m = hybrid()
    x = ids(2, 9)
    with torch.no_grad():
        whole = m(x)
        reset_net(m)
        parts = [m(x[:, :5])] + [m(x[:, t:t + 1]) for t in range(5, 9)]
        assert torch.allclose(torch.cat(parts, 1), whole, atol=1e-4)
        reset_net(m)
        alone = m(x[1:])
    assert torch.allclose(alone, whole[1:], atol=1e-4)
    assert sum(isinstance(b, CachedAttention) for b in m.modules()) == 2


def test_hybrid_select_goes_on_in_other_places():
    m = hybrid(2)
    x, more = ids(3, 6), ids(3, 2, seed=5)
    parents = [2, 0, 2]
    got = search(m, CPU, x, [(parents, more)])[:, 6:]
    with torch.no_grad():
        reset_net(m)
        want = m(torch.cat([x[parents], more], 1))[:, 6:]
    assert torch.allclose(got, want, atol=1e-4)


def test_hybrid_quantized():
    m = hybrid(3)
    x = ids(2, 5)
    want_model = dequantized(m)
    q = copy.deepcopy(m).quantize_()
    names = [n for n, b in q.named_modules() if isinstance(b, MX4Linear)]
    assert len(names) == 9 and "head" in names and not any(isinstance(b, nn.Linear) for b in q.modules())
    assert q.quantize_() is q
    with torch.no_grad():
        assert torch.allclose(q(x), want_model(x), atol=1e-4)
        reset_net(q)
        sf.optimize(q, sample_input=x, verbose=False)
        reset_net(q)
        reset_net(want_model)
        assert torch.allclose(q(x), want_model(x), atol=1e-4)


def test_models_without_attention_are_what_they_were():
    torch.manual_seed(0)
    a = spiking_ssm_tiny(vocab=8)
    assert not any(isinstance(b, (CachedAttention, MX4Linear)) for b in a.modules())
    with torch.no_grad():
        a(ids(2, 3, 8))
        a.select(torch.tensor([1, 1]))
        y = a(ids(2, 1, 8)[:1].expand(2, 1))
    assert torch.equal(y[0], y[1])


def test_select_of_nothing():
    check_select_of_nothing(CPU)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_hybrid_in_16_bits(dtype):
    check_hybrid_in_16_bits(CPU, dtype)


def test_saved_in_the_middle():
    check_saved(CPU)
