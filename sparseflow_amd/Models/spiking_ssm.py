"""A spiking state space model of token sequences: the example that runs the
state space operators with the spike-sparse Linear and the neurons.

Token time is the neurons' time: activations are [tokens, batch, dim], and every
LIF neuron integrates along the tokens.  A block is

    spikes = LIF(norm(residual))
    z, u, dt = in_proj(spikes)                   (a SparseLinear after optimize())
    x, B, C = silu(causal convolution of u)
    y = gated norm(selective scan(x, dt, B, C), z)
    residual += scale * norm(out_proj(LIF(y)))   (the second SparseLinear)

with the norm after a block, its residual scale and the next block's norm in one
pass.  With `attention_every`, every so many blocks one attends to all tokens before,
through a paged 4-bit cache, in the scan's place:

    q, k, v = in_proj(LIF(norm(residual)))
    residual += scale * norm(out_proj(LIF(attention(q, k, v))))

The model is stateful like its neurons: a forward continues the sequences of the last
one (a prompt, then its tokens one at a time) until reset_net(); select() lets the
sequences of a search go on in each other's places.  quantize_() keeps the projections
in the 4-bit format: the spikes that they read are exact in it."""

from __future__ import annotations

import torch
import torch.nn as nn

from ..neuron import BaseNode, LIFNode
from ..Ops._runtime import host_parents
from ..Ops.cached_attention import CachedAttention
from ..Ops.mx4_linear import quantize_linears_
from ..Ops.state_space import BlockNorm, CausalConv1d, SelectiveScan


def _lif(v_threshold: float) -> LIFNode:
    return LIFNode(tau=2.0, v_threshold=v_threshold, v_reset=0.0, detach_reset=True, step_mode="m")


class SpikingSSMBlock(nn.Module):
    """[tokens, batch, dim] -> the same, before the block's own norm."""

    def __init__(self, dim: int, head_dim: int = 64, state_dim: int = 64, groups: int = 1, expand: int = 2,
                 kernel_size: int = 4, v_threshold: float = 1.0):
        super().__init__()
        self.inner = expand * dim
        if self.inner % head_dim != 0:
            raise ValueError(f"expand * dim = {self.inner} must be divisible by head_dim={head_dim}")
        self.heads, self.head_dim, self.groups, self.state_dim = self.inner // head_dim, head_dim, groups, state_dim
        self.mixed = self.inner + 2 * groups * state_dim
        self.in_lif = _lif(v_threshold)
        # (The projection's width is rounded up to what the sparse Linear takes.)
        self.in_proj = nn.Linear(dim, -(-(self.inner + self.mixed + self.heads) // 4) * 4, bias=False)
        self.conv = CausalConv1d(self.mixed, kernel_size)
        self.scan = SelectiveScan(self.heads, head_dim, state_dim, groups)
        self.gate_norm = BlockNorm(self.inner, post=True, gate_first=True, group_size=self.inner // groups)
        self.out_lif = _lif(v_threshold)
        self.out_proj = nn.Linear(self.inner, dim, bias=False)

    def forward(self, h: torch.Tensor) -> torch.Tensor:
        t, b, _ = h.shape
        p = self.in_proj(self.in_lif(h).flatten(0, 1)).unflatten(0, (t, b))
        z, u, dt = p.split([self.inner, self.mixed, p.shape[-1] - self.inner - self.mixed], dim=-1)
        u = self.conv(u.transpose(0, 1))  # [batch, tokens, ...] from here
        gn = self.groups * self.state_dim
        x, B, C = u.split([self.inner, gn, gn], dim=-1)
        y = self.scan(x.unflatten(-1, (self.heads, self.head_dim)), dt[..., : self.heads].transpose(0, 1),
                      B.unflatten(-1, (self.groups, self.state_dim)), C.unflatten(-1, (self.groups, self.state_dim)))
        y, _ = self.gate_norm(y.flatten(-2).transpose(0, 1), gate=z)
        return self.out_proj(self.out_lif(y).flatten(0, 1)).unflatten(0, (t, b))


class SpikingAttentionBlock(nn.Module):
    """[tokens, batch, dim] -> the same, before the block's own norm."""

    def __init__(self, dim: int, head_dim: int = 64, kv_heads: int = 1, page_size: int = 64, v_threshold: float = 1.0):
        super().__init__()
        if dim % head_dim != 0 or dim // head_dim % kv_heads != 0:
            raise ValueError(f"dim={dim} must be a multiple of kv_heads={kv_heads} heads of head_dim={head_dim}")
        self.heads, self.kv_heads, self.head_dim = dim // head_dim, kv_heads, head_dim
        self.in_lif = _lif(v_threshold)
        self.in_proj = nn.Linear(dim, (self.heads + 2 * kv_heads) * head_dim, bias=False)
        self.attention = CachedAttention(page_size)
        self.out_lif = _lif(v_threshold)
        self.out_proj = nn.Linear(dim, dim, bias=False)

    def forward(self, h: torch.Tensor) -> torch.Tensor:
        t, b, _ = h.shape
        p = self.in_proj(self.in_lif(h).flatten(0, 1)).unflatten(0, (t, b)).transpose(0, 1)
        q, k, v = p.unflatten(-1, (-1, self.head_dim)).split([self.heads, self.kv_heads, self.kv_heads], dim=2)
        y = self.attention(q, k, v).flatten(-2).transpose(0, 1)
        return self.out_proj(self.out_lif(y).flatten(0, 1)).unflatten(0, (t, b))


class SpikingSSM(nn.Module):
    """ids [batch, tokens] -> logits [batch, tokens, vocab].  attention_every: block
    number attention_every, twice that and so on attend (0: none does)."""

    def __init__(self, vocab: int, dim: int = 192, depth: int = 4, head_dim: int = 64, state_dim: int = 64,
                 groups: int = 1, v_threshold: float = 1.0, attention_every: int = 0):
        super().__init__()
        self.vocab, self.dim = int(vocab), int(dim)
        self.embed = nn.Embedding(vocab, dim)
        self.first_norm = BlockNorm(dim, pre=True)
        self.blocks = nn.ModuleList(
            SpikingAttentionBlock(dim, head_dim, v_threshold=v_threshold)
            if attention_every and (i + 1) % attention_every == 0
            else SpikingSSMBlock(dim, head_dim, state_dim, groups, v_threshold=v_threshold) for i in range(depth))
        self.norms = nn.ModuleList(BlockNorm(dim, post=True, pre=True, scale=1.0) for _ in range(depth))
        self.head = nn.Linear(dim, vocab, bias=False)

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        r, h = self.first_norm(self.embed(ids.t()))
        for block, norm in zip(self.blocks, self.norms):
            r, h = norm(block(h), residual=r)
        return self.head(h).transpose(0, 1)

    def select(self, parents: torch.Tensor) -> None:
        """Sequence i of the batch becomes what sequence parents[i] was (a beam search's step)."""
        parents = parents.detach().cpu()
        for m in self.modules():
            if isinstance(m, BaseNode):
                if m.v is not None:
                    m.v = m.v.index_select(0, host_parents(parents, m.v.shape[0]).to(m.v.device))
            elif m is not self and hasattr(m, "select"):
                m.select(parents)

    def quantize_(self) -> "SpikingSSM":
        """The projections' weights to 4 bits, with the spikes that the blocks' read."""
        quantize_linears_(self.blocks, quantize_input=True)
        quantize_linears_(self, only=lambda name, _: name == "head")
        return self


def spiking_ssm_tiny(vocab: int = 256, v_threshold: float = 1.0) -> SpikingSSM:
    """Width 192 (6 heads of 64 inside the blocks), four blocks."""
    return SpikingSSM(vocab, 192, 4, 64, 64, 1, v_threshold)


def spiking_ssm_hybrid_tiny(vocab: int = 256, v_threshold: float = 1.0) -> SpikingSSM:
    """The same with attention (3 heads of 64, keys and values in one) in every second block."""
    return SpikingSSM(vocab, 192, 4, 64, 64, 1, v_threshold, attention_every=2)


MODEL_BUILDERS = {"spiking_ssm_tiny": spiking_ssm_tiny, "spiking_ssm_hybrid_tiny": spiking_ssm_hybrid_tiny}
