"""The state space operators in 64 bits on the CPU, from their definitions: the
causal convolution, the selective scan and the block norm.  Next to each result
comes its magnitude, the same sum over absolute values, that error bounds are
multiples of."""

from __future__ import annotations

import torch

F64 = torch.float64


def spans(total: int, batch: int, offsets):
    """(first row, rows) of each sequence of a packed batch."""
    at = [min(max(int(v), 0), total) for v in offsets]
    return [(a, max(0, b - a)) for a, b in zip(at, at[1:])]


def silu(v):
    return v * torch.sigmoid(v)


def conv1d(x, weight, bias, act, before):
    """One sequence: x [n, C], weight [C, K], before [K - 1, C] -> (y, state, magnitude of y)."""
    x, w = x.to(F64), weight.to(F64)
    k = w.shape[1]
    u = torch.cat([before.to(F64), x])
    y = torch.zeros(x.shape, dtype=F64)
    mag = torch.zeros(x.shape, dtype=F64)
    for i in range(k):
        y += w[:, i] * u[i:i + x.shape[0]]
        mag += (w[:, i] * u[i:i + x.shape[0]]).abs()
    if bias is not None:
        y += bias.to(F64)
        mag += bias.to(F64).abs()
    return (silu(y) if act == "silu" else y), u[x.shape[0]:], mag


def scan(x, dt, A, B, C, D, dt_bias, softplus, h0):
    """One sequence: x [n, H, P], dt [n, H], B, C [n, G, N], h0 [H, P, N] ->
    (y, state, magnitude of y, magnitude of the state)."""
    x, dt, A, B, C = (t.to(F64) for t in (x, dt, A, B, C))
    r = x.shape[1] // B.shape[1]
    h = h0.to(F64).clone()
    hm = h.abs()
    y = torch.zeros(x.shape, dtype=F64)
    ym = torch.zeros(x.shape, dtype=F64)
    for t in range(x.shape[0]):
        d = dt[t] if dt_bias is None else dt[t] + dt_bias.to(F64)
        if softplus:
            d = torch.logaddexp(d, torch.zeros((), dtype=F64))
        a = torch.exp(A * d)[:, None, None]
        b, c = B[t].repeat_interleave(r, 0)[:, None, :], C[t].repeat_interleave(r, 0)[:, None, :]
        u = (d[:, None] * x[t])[:, :, None]
        h = a * h + u * b
        hm = a * hm + (u * b).abs()
        y[t] = (h * c).sum(-1)
        ym[t] = (hm * c.abs()).sum(-1)
        if D is not None:
            y[t] += D.to(F64)[:, None] * x[t]
            ym[t] += (D.to(F64)[:, None] * x[t]).abs()
    return y, h, ym, hm


def block_norm(x, gate, act, gate_first, post, group, residual, scale, pre, eps):
    """Rows [..., dim] -> (r, h or None, magnitude of r)."""
    def rms(t, w, size):
        g = t.reshape(t.shape[:-1] + (-1, size))
        return (g / torch.sqrt(g.square().mean(-1, keepdim=True) + eps)).reshape(t.shape) * w.to(F64)

    t = x.to(F64)
    if gate is not None:
        g = gate.to(F64)
        g = silu(g) if act == "silu" else torch.sigmoid(g) if act == "sigmoid" else g
    if gate is not None and gate_first:
        t = t * g
    if post is not None:
        t = rms(t, post, group)
    if gate is not None and not gate_first:
        t = t * g
    if scale is not None:
        t = t * (scale.to(F64) if isinstance(scale, torch.Tensor) else scale)
    mag = t.abs()
    if residual is not None:
        t = t + residual.to(F64)
        mag = mag + residual.to(F64).abs()
    return t, None if pre is None else rms(t, pre, t.shape[-1]), mag
