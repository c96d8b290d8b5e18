"""MX4Linear: a Linear whose weight is kept in the microscaled 4-bit format
(Kernels/mx4.py): 17 bytes for 32 weights.

Inputs of shape [..., in_features] are taken as they are, or, with `quantize_input`,
brought to the format first, which runs the 4-bit matrix instructions.  Spikes lose
nothing by that: a block of zeros and ones is exact in the format.  The weight is a
buffer (the format has no gradients); inference only."""

from __future__ import annotations

from typing import Callable, Optional

import torch
import torch.nn as nn

from ..Kernels.mx4 import blocks_of, mx4_dequantize, mx4_linear_forward, mx4_quantize
from ._runtime import WeightLayout


def _float32(bias: torch.Tensor) -> torch.Tensor:
    return bias.detach().float().contiguous()


class MX4Linear(nn.Module):
    def __init__(self, in_features: int, out_features: int, bias: bool = True, quantize_input: bool = False,
                 device=None):
        super().__init__()
        self.in_features, self.out_features, self.quantize_input = int(in_features), int(out_features), bool(quantize_input)
        n = blocks_of(self.in_features)
        self.register_buffer("codes", torch.zeros(self.out_features, 16 * n, dtype=torch.uint8, device=device))
        self.register_buffer("scales", torch.zeros(self.out_features, n, dtype=torch.uint8, device=device))
        self.register_buffer("bias", torch.zeros(self.out_features, device=device) if bias else None)
        self._bias = WeightLayout(_float32)

    @classmethod
    def from_dense(cls, linear: nn.Linear, quantize_input: bool = False) -> "MX4Linear":
        """Of a module with an nn.Linear's weight and bias (a SparseLinear too)."""
        w, b = linear.weight.detach(), linear.bias
        mod = cls(w.shape[1], w.shape[0], b is not None, quantize_input, w.device)
        mod.codes, mod.scales = mx4_quantize(w)
        if b is not None:
            mod.bias.copy_(b.detach())
        return mod.train(linear.training)

    def dequantized_weight(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return mx4_dequantize(self.codes, self.scales, self.in_features, dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() < 1 or x.shape[-1] != self.in_features:
            raise ValueError(f"MX4Linear takes [..., {self.in_features}] input, not {tuple(x.shape)}")
        bias: Optional[torch.Tensor] = self.bias
        if bias is not None and bias.dtype != torch.float32:
            bias = self._bias(bias)
        dtype = x.dtype
        return mx4_linear_forward(mx4_quantize(x) if self.quantize_input else x, (self.codes, self.scales), bias, dtype)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, "
                f"quantize_input={self.quantize_input}")


def quantize_linears_(net: nn.Module, quantize_input: bool = False,
                      only: Optional[Callable[[str, nn.Module], bool]] = None) -> int:
    """Replaces the nn.Linear and SparseLinear modules of `net` (those that only(name,
    module) picks) by MX4Linear -> how many.  Subclasses stay: their forward may be another,
    or their owner read the weight by itself (nn.MultiheadAttention).  Hooks are the old
    module's, as everywhere that modules are replaced."""
    from .sparse_linear import SparseLinear

    found = [(name, m) for name, m in net.named_modules(remove_duplicate=False)
             if name and type(m) in (nn.Linear, SparseLinear) and (only is None or only(name, m))]
    made = {}  # (a module that stands in two places is one afterwards too)
    for _, m in found:
        if m not in made:
            made[m] = MX4Linear.from_dense(m, quantize_input)
    for name, m in found:
        parent, _, leaf = name.rpartition(".")
        setattr(net.get_submodule(parent), leaf, made[m])
    return len(found)
