"""Modules over the 4-bit operators on the GPU, and the model that runs them together."""

import copy

import pytest
import torch

from sparseflow_amd import _lib
from sparseflow_amd.Ops import CachedAttention
from tests.gpu_helpers import DEV, announce, native_loaded
from tests.mx4_module_checks import check_cached_attention, check_hybrid_in_16_bits, check_linear_module, \
    check_saved, check_select, check_select_of_nothing, hybrid, ids, search

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias,quantize_input,sparse", [(True, False, False), (False, True, False), (True, True, True)])
def test_linear_module(dtype, bias, quantize_input, sparse):
    check_linear_module(DEV, dtype, bias, quantize_input, sparse)
    assert native_loaded()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,parts", [(1, [3, 1, 2]), (4, [7, 1, 1, 5, 1]), (64, [1, 1, 170])])
def test_cached_attention_module(page, parts, dtype):
    announce(f"cached attention module {page} {parts} {dtype}")
    check_cached_attention(DEV, dtype, page, parts)


@pytest.mark.parametrize("page,before,after", [(4, 8, 1), (4, 6, 3), (1, 2, 1), (16, 5, 12), (64, 700, 1)])
def test_select(page, before, after):
    announce(f"select {page} {before} {after}")
    check_select(DEV, page, before, after)


def test_refused_calls_leave_the_sequences():
    mod = CachedAttention(page_size=4)
    k = torch.randn(2, 3, 2, 8, device=DEV)
    mod(k, k, k)
    for args in ((k, k.half(), k), (k.cpu(), k, k), (k, k, k[:, :2])):
        with pytest.raises(ValueError):
            mod(*args)
    with pytest.raises(ValueError):
        mod.select(torch.tensor([0, 2], device=DEV))
    assert mod.state.tokens == 3


def _logits_agree(got, want):
    """The neurons' thresholds apart both sides differ by float32 rounding; of the few thousand neuron steps, each within
    1e-6 of its threshold with a chance of about 1e-6, none is expected to fall to the other side."""
    assert torch.isfinite(got).all()
    off = (got - want).abs().amax(-1)
    assert bool((off < 1e-3).all()), f"{int((off >= 1e-3).sum())} of {off.numel()} positions differ, most {float(off.max()):.3g}"


@pytest.mark.parametrize("quantized", [False, True])
def test_hybrid_search_matches_the_host(quantized):
    """Prompts, then steps of a search whose sequences go on in each other's places."""
    announce(f"hybrid search quantized={quantized}")
    host = hybrid(7)
    if quantized:
        host.quantize_()
    dev = copy.deepcopy(host).to(DEV)
    prompt = ids(3, 21)
    steps = [([2, 0, 2], ids(3, 1, seed=2)), ([1, 1, 0], ids(3, 1, seed=3)), ([0, 1, 2], ids(3, 2, seed=4))]
    want = search(host, torch.device("cpu"), prompt, steps)
    _lib.timing_reset()
    _lib.timing_enable(True)
    got = search(dev, DEV, prompt, steps)
    torch.cuda.synchronize()
    stats = _lib.timing_collect()
    _lib.timing_enable(False)
    launched = {n for n, (c, _) in stats.items() if c}
    assert {"mx4_append", "mx4_attention", "pages"} <= launched, launched
    assert not quantized or {"mx4_quantize", "mx4_linear"} <= launched, launched
    _logits_agree(got, want)


def test_select_of_nothing():
    check_select_of_nothing(DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_hybrid_in_16_bits(dtype):
    check_hybrid_in_16_bits(DEV, dtype)


def test_saved_in_the_middle():
    check_saved(DEV)
