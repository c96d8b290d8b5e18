"""nn.Modules over the state space operators: the short causal convolution, the
selective scan and the block norm.

CausalConv1d and SelectiveScan are stateful like the neurons (neuron.py): a
forward continues each sequence from where the last one left it, in state rows of
their own, until reset().  A prompt of one token runs the single-token kernels.
Parameters of another type than the kernels' float32 (a model in 16 bits) are cast
when they change.  Inference only."""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn as nn

from ..Kernels.block_norm import block_norm_forward
from ..Kernels.causal_conv1d import causal_conv1d_forward, causal_conv1d_step
from ..Kernels.selective_scan import selective_scan_forward, selective_scan_step
from ._runtime import WeightLayout, host_parents


def _cast(param: torch.Tensor) -> torch.Tensor:
    return param.detach().float().contiguous()


def _decay_rates(log: torch.Tensor) -> torch.Tensor:
    return -torch.exp(log.detach().float())


class _Float32:
    """A parameter as the kernels take it."""

    def __init__(self):
        self._cast = WeightLayout(_cast)

    def __call__(self, param: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
        return param if param is None or (param.dtype == torch.float32 and param.is_contiguous()) else self._cast(param)


class _Stateful(nn.Module):
    def __init__(self):
        super().__init__()
        self.state: Optional[torch.Tensor] = None

    def reset(self):
        self.state = None

    def select(self, parents: torch.Tensor) -> None:
        """Sequence i becomes what sequence parents[i] was (integers [batch])."""
        if self.state is not None:
            self.state = self.state.index_select(0, host_parents(parents, self.state.shape[0]).to(self.state.device))

    def _state_for(self, shape: Tuple[int, ...], dtype: torch.dtype, device: torch.device) -> Optional[torch.Tensor]:
        """The kept state, if it is one for such a batch (as the neurons decide)."""
        s = self.state
        return s if s is not None and tuple(s.shape) == shape and s.dtype == dtype and s.device == device else None


class CausalConv1d(_Stateful):
    """x [batch, tokens, channels] -> the same (Kernels/causal_conv1d.py)."""

    def __init__(self, channels: int, kernel_size: int = 4, bias: bool = True, activation: Optional[str] = "silu"):
        super().__init__()
        self.channels, self.kernel_size, self.activation = int(channels), int(kernel_size), activation
        self.weight = nn.Parameter(torch.empty(self.channels, self.kernel_size))
        self.bias = nn.Parameter(torch.zeros(self.channels)) if bias else None
        nn.init.uniform_(self.weight, -self.kernel_size ** -0.5, self.kernel_size ** -0.5)
        self._weight, self._bias = _Float32(), _Float32()

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        state = self._state_for((x.shape[0], self.kernel_size - 1, self.channels), x.dtype, x.device)
        weight, bias = self._weight(self.weight), self._bias(self.bias)
        if state is not None and x.shape[1] == 1:
            return causal_conv1d_step(state, x[:, 0], weight, bias, activation=self.activation)[:, None]
        y, self.state = causal_conv1d_forward(x, weight, bias, activation=self.activation, initial_state=state,
                                              final_state=state)
        return y

    def extra_repr(self) -> str:
        return f"channels={self.channels}, kernel_size={self.kernel_size}, activation={self.activation}"


class SelectiveScan(_Stateful):
    """x [batch, tokens, heads, head_dim], dt [..., heads], B and C [..., groups,
    state_dim] -> y like x (Kernels/selective_scan.py).  The decay rates are
    -exp(A_log); dt_bias starts with step sizes between 0.001 and 0.1."""

    def __init__(self, heads: int, head_dim: int, state_dim: int, groups: int = 1):
        super().__init__()
        if heads % groups != 0:
            raise ValueError(f"groups={groups} does not divide heads={heads}")
        self.heads, self.head_dim, self.state_dim, self.groups = int(heads), int(head_dim), int(state_dim), int(groups)
        step = torch.exp(torch.empty(self.heads).uniform_(math.log(1e-3), math.log(1e-1)))
        self.A_log = nn.Parameter(torch.log(torch.empty(self.heads).uniform_(1.0, 16.0)))
        self.D = nn.Parameter(torch.ones(self.heads))
        self.dt_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self._rates = WeightLayout(_decay_rates)
        self._D, self._dt_bias = _Float32(), _Float32()

    def forward(self, x: torch.Tensor, dt: torch.Tensor, B: torch.Tensor, C: torch.Tensor) -> torch.Tensor:
        A, D, dt_bias = self._rates(self.A_log), self._D(self.D), self._dt_bias(self.dt_bias)
        state = self._state_for((x.shape[0], self.heads, self.head_dim, self.state_dim), torch.float32, x.device)
        if state is not None and x.shape[1] == 1:
            return selective_scan_step(state, x[:, 0], dt[:, 0], A, B[:, 0], C[:, 0], D=D, dt_bias=dt_bias)[:, None]
        y, self.state = selective_scan_forward(x, dt, A, B, C, D=D, dt_bias=dt_bias, initial_state=state, final_state=state)
        return y

    def extra_repr(self) -> str:
        return (f"heads={self.heads}, head_dim={self.head_dim}, state_dim={self.state_dim}, groups={self.groups}")


class BlockNorm(nn.Module):
    """(r, h) of Kernels/block_norm.py with the weights that are asked for: post
    (the norm of the block's output, over group_size columns), scale (of the
    residual branch, per column) and pre (the next block's norm)."""

    def __init__(self, dim: int, post: bool = False, pre: bool = False, scale: Optional[float] = None,
                 group_size: Optional[int] = None, gate_first: bool = False, activation: Optional[str] = "silu",
                 eps: float = 1e-5):
        super().__init__()
        self.dim, self.group_size, self.gate_first, self.activation, self.eps = int(dim), group_size, gate_first, activation, eps
        self.post_weight = nn.Parameter(torch.ones(self.dim)) if post else None
        self.pre_weight = nn.Parameter(torch.ones(self.dim)) if pre else None
        self.scale = nn.Parameter(torch.full((self.dim,), float(scale))) if scale is not None else None
        self._post, self._pre, self._scale = _Float32(), _Float32(), _Float32()

    def forward(self, x: torch.Tensor, gate: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None
                ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        return block_norm_forward(x, gate=gate, activation=self.activation, gate_first=self.gate_first,
                                  post_weight=self._post(self.post_weight), group_size=self.group_size, residual=residual,
                                  scale=self._scale(self.scale), pre_weight=self._pre(self.pre_weight), eps=self.eps)

    def extra_repr(self) -> str:
        return f"dim={self.dim}, group_size={self.group_size}, gate_first={self.gate_first}, eps={self.eps}"
