"""Short causal convolution over the token axis, one filter per channel:

    y[t, c] = act(bias[c] + sum_k weight[c, k] * u[t - K + 1 + k, c])

u is x, and before a sequence's first token its state: the K - 1 inputs read
before it (oldest first), or zeros.  `causal_conv1d_forward` takes prompts,
`causal_conv1d_step` one token of each sequence with the states in a pool.
Device tensors run sf_causal_conv1d / sf_causal_conv1d_step; host tensors the
torch form below (the checker too).  Sums are float32.  Inference only: nothing
is recorded for a backward pass."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _lib
from ._sequences import Plans, check_apart, check_index, check_input, check_like, check_out, check_param, check_pool, \
    host_slots, host_spans, last_contiguous, signature

_prompts, _steps = Plans(), Plans()


def _check(x: torch.Tensor, weight: torch.Tensor, bias, activation) -> Tuple[int, int]:
    check_input(x, "x")
    ch = int(x.shape[-1])
    if weight.dim() != 2 or weight.shape[1] < 1 or ch < 1:
        raise ValueError(f"weight is {tuple(weight.shape)}: ({ch}, kernel) is wanted")
    k = int(weight.shape[1])
    check_param(weight, x, "weight", (ch, k))
    check_param(bias, x, "bias", (ch,))
    if activation not in (None, "silu"):
        raise ValueError(f"activation is {activation!r}: None or 'silu' is wanted")
    if k > 8:
        raise _lib.UnsupportedError(f"kernel {k} is over 8")
    return ch, k


def _host_conv(u: torch.Tensor, weight: torch.Tensor, bias, activation) -> torch.Tensor:
    """u [K - 1 + tokens, C] -> [tokens, C] in float32."""
    k = weight.shape[1]
    n = u.shape[0] - (k - 1)
    y = torch.zeros(n, u.shape[1]) if bias is None else bias.expand(n, -1).clone()
    for i in range(k):
        y += weight[:, i] * u[i:i + n].float()
    return y / (1 + torch.exp(-y)) if activation == "silu" else y


def causal_conv1d_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                          activation: Optional[str] = None, initial_state: Optional[torch.Tensor] = None,
                          offsets: Optional[torch.Tensor] = None, max_len: Optional[int] = None,
                          slots: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                          final_state: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [batch, tokens, C], or [total, C] with offsets -> (y, final state).

    weight float32 [C, K <= 8], bias float32 [C]; activation None or "silu".
    initial_state, final_state [batch, K - 1, C] in x's type, or pools
    [rows, K - 1, C] with slots (int32 [batch]; a slot outside the pool: zeros
    before, nothing kept); they may be one tensor.  max_len, the longest
    sequence, sizes the launch of a packed call (default: all its tokens).  Apart
    from that, what is written shares no memory with what is read.
    """
    if x.is_cuda:
        x = last_contiguous(x)
    if max_len is not None:
        max_len = int(max_len)
    key = (signature(x, weight, bias, initial_state, offsets, slots, out, final_state), activation, max_len)
    plan = _prompts.get(key) or _prompts.make(key, _check_prompt, x, weight, bias, activation, initial_state, offsets,
                                              max_len, slots, out, final_state)
    shape, desc = plan
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        check_apart(out, "out", {"x": x, "initial_state": initial_state, "final_state": final_state})
    if final_state is None:
        final_state = torch.empty(shape, dtype=x.dtype, device=x.device)
    else:
        check_apart(final_state, "final_state", {"x": x} if final_state is initial_state else
                    {"x": x, "initial_state": initial_state}, same=("initial_state",))
    if not x.is_cuda:
        with torch.no_grad():
            keep = shape[1]
            rows = host_slots(shape[0], final_state.shape[0], slots)
            for b, (xs, ys) in enumerate(zip(host_spans(x, offsets), host_spans(out, offsets))):
                before = initial_state[rows[b]] if initial_state is not None and rows[b] >= 0 \
                    else x.new_zeros(keep, x.shape[-1])
                u = torch.cat([before, xs])
                ys.copy_(_host_conv(u, weight, bias, activation))
                if rows[b] >= 0:
                    final_state[rows[b]] = u[u.shape[0] - keep:]
            return out, final_state
    _lib.causal_conv1d(desc, x, weight, bias, offsets, slots, initial_state, out, final_state)
    return out, final_state


def _check_prompt(x, weight, bias, activation, initial_state, offsets, max_len, slots, out, final_state):
    """-> (the states' shape, the descriptor of a device call)."""
    if x.dim() != (3 if offsets is None else 2):
        raise ValueError(f"x is {tuple(x.shape)}: (batch, tokens, C), or (total, C) with offsets, is wanted")
    ch, k = _check(x, weight, bias, activation)
    if offsets is not None and offsets.numel() < 1:
        raise ValueError("offsets is empty: one more than the sequences is wanted")
    batch = int(x.shape[0]) if offsets is None else int(offsets.numel()) - 1
    tokens = int(x.shape[-2])
    check_index(offsets, x, "offsets", batch + 1)
    check_index(slots, x, "slots", batch)
    check_pool(initial_state, x, "initial_state", (k - 1, ch), x.dtype, batch, slots)
    check_pool(final_state, x, "final_state", (k - 1, ch), x.dtype, batch, slots)
    if slots is not None and final_state is None:
        raise ValueError("slots without final_state: the pool that keeps the states is wanted")
    if initial_state is not None and final_state is not None and initial_state.shape != final_state.shape:
        raise ValueError("initial_state and final_state have different numbers of rows")
    if out is not None:
        check_like(out, x, "out", tuple(x.shape))
        check_out(out, "out")
        if out.stride(-1) != 1 and ch > 1:
            raise ValueError("out: a contiguous last axis is wanted")
    if not x.is_cuda:
        return (batch, k - 1, ch), None
    rows = batch if final_state is None else int(final_state.shape[0])
    # (A new out has the default strides.)
    ys = torch.empty(x.shape, device="meta").stride() if out is None else out.stride()
    if offsets is None:
        longest, xs, ys = tokens, x.stride()[:2], ys[:2]
    else:
        longest = tokens if max_len is None else min(max(int(max_len), 0), tokens)
        xs, ys = (0, x.stride(0)), (0, ys[0])
    return (rows, k - 1, ch), _lib.conv1d_desc(batch, tokens, longest, rows, xs, ys, ch, k, x.dtype, activation)


def causal_conv1d_step(state: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                       bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                       slots: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of each sequence: x [batch, C] -> y [batch, C].

    state [batch, K - 1, C] in x's type, or a pool [rows, K - 1, C] with slots
    (int32 [batch], no two alike), moves on by the token in place.  A slot
    outside the pool: y is zero there and no state changes.  out may be x.
    """
    if x.is_cuda:
        x = last_contiguous(x)
    key = (signature(state, x, weight, bias, slots, out), activation)
    plan = _steps.get(key) or _steps.make(key, _check_step, state, x, weight, bias, activation, slots, out)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        check_apart(out, "out", {"x": x, "state": state}, same=("x",))
    if not x.is_cuda:
        with torch.no_grad():
            for b, row in enumerate(host_slots(x.shape[0], state.shape[0], slots)):
                if row < 0:
                    out[b] = 0
                    continue
                u = torch.cat([state[row], x[b:b + 1]])
                out[b] = _host_conv(u, weight, bias, activation)[0].to(x.dtype)
                state[row] = u[1:]
            return out
    _lib.causal_conv1d_step(plan[0], state, x, weight, bias, slots, out)
    return out


def _check_step(state, x, weight, bias, activation, slots, out):
    """-> (the descriptor of a device call,)."""
    if x.dim() != 2:
        raise ValueError(f"x is {tuple(x.shape)}: (batch, C) is wanted")
    ch, k = _check(x, weight, bias, activation)
    batch = int(x.shape[0])
    check_index(slots, x, "slots", batch)
    check_pool(state, x, "state", (k - 1, ch), x.dtype, batch, slots)
    if out is not None:
        check_like(out, x, "out", (batch, ch))
        check_out(out, "out")
        if out.stride(-1) != 1 and ch > 1:
            raise ValueError("out: a contiguous last axis is wanted")
    if not x.is_cuda:
        return (None,)
    ys = ch if out is None else out.stride(0)
    return (_lib.conv1d_desc(batch, 1, 1, int(state.shape[0]), (x.stride(0), 0), (ys, 0), ch, k, x.dtype, activation),)
