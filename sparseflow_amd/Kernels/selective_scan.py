"""Selective state space scan: the leaky integrator of a neuron with a decay
that the input sets and a matrix for its state.  Per sequence and head, with
d_t = softplus(dt_t + dt_bias),

    h_t = exp(A d_t) h_{t-1} + d_t x_t (outer) B_t        [head_dim, state_dim]
    y_t = h_t C_t + D x_t                                 [head_dim]

`selective_scan_forward` takes prompts, `selective_scan_step` one token of each
sequence with the states in a pool.  Device tensors run sf_selective_scan /
sf_selective_scan_step; host tensors the torch form below (the checker too).
States and sums are float32.  Inference only: nothing is recorded for a
backward pass."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _lib
from ._sequences import Plans, check_apart, check_index, check_input, check_like, check_out, check_param, check_pool, \
    host_slots, host_spans, last_contiguous, signature

_prompts, _steps = Plans(), Plans()


def _check(x, dt, A, B, C, D, dt_bias) -> Tuple[int, int, int, int]:
    """x [..., H, P], dt [..., H], B and C [..., G, N] -> H, P, G, N."""
    check_input(x, "x")
    lead, H, P = tuple(x.shape[:-2]), int(x.shape[-2]), int(x.shape[-1])
    if B.dim() != x.dim():
        raise ValueError(f"B is {tuple(B.shape)}: {lead} + (groups, state_dim) is wanted")
    G, N = int(B.shape[-2]), int(B.shape[-1])
    if min(H, P, G, N) < 1 or H % G != 0:
        raise ValueError(f"x {tuple(x.shape)} and B {tuple(B.shape)}: groups that divide the heads are wanted")
    check_like(dt, x, "dt", lead + (H,))
    check_like(B, x, "B", lead + (G, N))
    check_like(C, x, "C", lead + (G, N))
    if A is None:
        raise ValueError(f"A: a contiguous ({H},) float32 is wanted")
    check_param(A, x, "A", (H,))
    check_param(D, x, "D", (H,))
    check_param(dt_bias, x, "dt_bias", (H,))
    if N > 256:
        raise _lib.UnsupportedError(f"state_dim {N} is over 256")
    return H, P, G, N


def _host_token(h, x, dt, A, B, C, D, dt_bias, dt_softplus):
    """One token of one sequence in float32: h [H, P, N] is updated, y [H, P]."""
    d = dt.float() if dt_bias is None else dt.float() + dt_bias
    if dt_softplus:
        d = torch.clamp(d, min=0) + torch.log1p(torch.exp(-d.abs()))
    r = x.shape[0] // B.shape[0]
    b, c = (t.float().repeat_interleave(r, 0)[:, None] for t in (B, C))
    h.mul_(torch.exp(A * d)[:, None, None]).add_((d[:, None] * x.float())[..., None] * b)
    y = (h * c).sum(-1)
    return y if D is None else y + D[:, None] * x.float()


def selective_scan_forward(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor,
                           D: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                           dt_softplus: bool = True, initial_state: Optional[torch.Tensor] = None,
                           offsets: Optional[torch.Tensor] = None, max_len: Optional[int] = None,
                           slots: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                           final_state: Optional[torch.Tensor] = None,
                           workspace: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [batch, tokens, H, P], or [total, H, P] with offsets -> (y, final state).

    dt [..., H], B and C [..., G, N] in x's type (any strides over a contiguous
    last axis: views of one projection's output are read in place); A, D,
    dt_bias float32 [H]; G divides H, N <= 256.  initial_state, final_state
    float32 [batch, H, P, N], or pools [rows, H, P, N] with slots (int32
    [batch]; a slot outside the pool: a zero state, not kept); they may be one
    tensor.  max_len, the longest sequence, sizes the launch of a packed call
    (default: all its tokens).  workspace optionally holds the scratch between
    calls (contiguous, uint8; a new one where it is too small).  Apart from the
    states, what is written shares no memory with what is read.
    """
    if x.is_cuda:
        x, B, C = last_contiguous(x), last_contiguous(B), last_contiguous(C)
    if max_len is not None:
        max_len = int(max_len)
    dt_softplus = bool(dt_softplus)
    key = (signature(x, dt, A, B, C, D, dt_bias, offsets, slots, initial_state, out, final_state), max_len, dt_softplus)
    plan = _prompts.get(key) or _prompts.make(key, _check_prompt, x, dt, A, B, C, D, dt_bias, dt_softplus, initial_state,
                                              offsets, max_len, slots, out, final_state)
    shape, desc = plan
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        check_apart(out, "out", {"x": x, "dt": dt, "B": B, "C": C, "initial_state": initial_state, "final_state": final_state})
    if final_state is None:
        final_state = torch.empty(shape, dtype=torch.float32, device=x.device)
    elif final_state is not initial_state:
        check_apart(final_state, "final_state", {"x": x, "dt": dt, "B": B, "C": C, "initial_state": initial_state},
                    same=("initial_state",))
    if workspace is not None and not workspace.is_contiguous():
        raise ValueError(f"workspace has strides {tuple(workspace.stride())}: a contiguous one is wanted")
    if not x.is_cuda:
        with torch.no_grad():
            H, P, N = shape[1:]
            rows = host_slots(shape[0], final_state.shape[0], slots)
            spans = zip(*(host_spans(t, offsets) for t in (x, dt, B, C, out)))
            for b, (xs, ds, bs, cs, ys) in enumerate(spans):
                h = torch.zeros(H, P, N) if initial_state is None or rows[b] < 0 else initial_state[rows[b]].clone()
                for t in range(xs.shape[0]):
                    ys[t] = _host_token(h, xs[t], ds[t], A, bs[t], cs[t], D, dt_bias, dt_softplus).to(x.dtype)
                if rows[b] >= 0:
                    final_state[rows[b]] = h
            return out, final_state
    need = desc[2]
    if need == 0:
        workspace = None
    elif workspace is None or workspace.device != x.device or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    _lib.selective_scan(desc, x, dt, A, B, C, D, dt_bias, offsets, slots, initial_state, out, final_state, workspace)
    return out, final_state


def _check_prompt(x, dt, A, B, C, D, dt_bias, dt_softplus, initial_state, offsets, max_len, slots, out, final_state):
    """-> (the states' shape, the descriptor of a device call)."""
    if x.dim() != (4 if offsets is None else 3):
        raise ValueError(f"x is {tuple(x.shape)}: (batch, tokens, H, P), or (total, H, P) with offsets, is wanted")
    H, P, G, N = _check(x, dt, A, B, C, D, dt_bias)
    if offsets is not None and offsets.numel() < 1:
        raise ValueError("offsets is empty: one more than the sequences is wanted")
    batch = int(x.shape[0]) if offsets is None else int(offsets.numel()) - 1
    tokens = int(x.shape[-3])
    check_index(offsets, x, "offsets", batch + 1)
    check_index(slots, x, "slots", batch)
    check_pool(initial_state, x, "initial_state", (H, P, N), torch.float32, batch, slots)
    check_pool(final_state, x, "final_state", (H, P, N), torch.float32, batch, slots)
    if slots is not None and final_state is None:
        raise ValueError("slots without final_state: the pool that keeps the states is wanted")
    if initial_state is not None and final_state is not None and initial_state.shape != final_state.shape:
        raise ValueError("initial_state and final_state have different numbers of rows")
    if out is not None:
        check_like(out, x, "out", tuple(x.shape))
        check_out(out, "out")
        if out.stride(-1) != 1 and P > 1:
            raise ValueError("out: a contiguous last axis is wanted")
    shape = (batch, H, P, N) if final_state is None else tuple(final_state.shape)
    if not x.is_cuda:
        return (batch, H, P, N), None
    # (A new out has the default strides.)
    ys = torch.empty(x.shape, device="meta").stride() if out is None else out.stride()
    if offsets is None:
        longest = tokens
        strides = (x.stride()[:3], dt.stride(), B.stride()[:3], C.stride()[:3], ys[:3])
    else:
        longest = tokens if max_len is None else min(max(int(max_len), 0), tokens)
        strides = ((0,) + x.stride()[:2], (0,) + dt.stride(), (0,) + B.stride()[:2], (0,) + C.stride()[:2],
                   (0,) + ys[:2])
    return shape, _lib.scan_desc(batch, tokens, longest, shape[0], *strides, H, P, G, N, x.dtype, bool(dt_softplus))


def selective_scan_step(state: torch.Tensor, x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                        C: torch.Tensor, D: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                        dt_softplus: bool = True, slots: Optional[torch.Tensor] = None,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token of each sequence: x [batch, H, P] -> y [batch, H, P].

    dt [batch, H], B and C [batch, G, N]; state float32 [batch, H, P, N], or a
    pool [rows, H, P, N] with slots (int32 [batch], no two alike), moves on by
    the token in place.  A slot outside the pool: y is zero there and no state
    changes.  out may be x.
    """
    if x.is_cuda:
        x, B, C = last_contiguous(x), last_contiguous(B), last_contiguous(C)
    dt_softplus = bool(dt_softplus)
    key = (signature(state, x, dt, A, B, C, D, dt_bias, slots, out), dt_softplus)
    plan = _steps.get(key) or _steps.make(key, _check_step, state, x, dt, A, B, C, D, dt_bias, dt_softplus, slots, out)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        check_apart(out, "out", {"x": x, "dt": dt, "B": B, "C": C, "state": state}, same=("x",))
    if not x.is_cuda:
        with torch.no_grad():
            for b, row in enumerate(host_slots(x.shape[0], state.shape[0], slots)):
                if row < 0:
                    out[b] = 0
                else:
                    out[b] = _host_token(state[row], x[b], dt[b], A, B[b], C[b], D, dt_bias, dt_softplus).to(x.dtype)
            return out
    _lib.selective_scan_step(plan[0], state, x, dt, A, B, C, D, dt_bias, slots, out)
    return out


def _check_step(state, x, dt, A, B, C, D, dt_bias, dt_softplus, slots, out):
    """-> (the descriptor of a device call,)."""
    if x.dim() != 3:
        raise ValueError(f"x is {tuple(x.shape)}: (batch, H, P) is wanted")
    H, P, G, N = _check(x, dt, A, B, C, D, dt_bias)
    batch = int(x.shape[0])
    check_index(slots, x, "slots", batch)
    check_pool(state, x, "state", (H, P, N), torch.float32, batch, slots)
    if out is not None:
        check_like(out, x, "out", (batch, H, P))
        check_out(out, "out")
        if out.stride(-1) != 1 and P > 1:
            raise ValueError("out: a contiguous last axis is wanted")
    if not x.is_cuda:
        return (None,)
    pair = lambda s: (s[0], 0, s[1])  # noqa: E731
    ys = (H * P, P) if out is None else out.stride()
    return (_lib.scan_desc(batch, 1, 1, int(state.shape[0]), pair(x.stride()), pair(dt.stride()), pair(B.stride()),
                           pair(C.stride()), pair(ys), H, P, G, N, x.dtype, bool(dt_softplus)),)
