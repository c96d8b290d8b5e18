"""The norms around a block with its gate and residual scale, in one pass:

    t = x;  gate_first: t *= act(gate)
    post_weight:  t *= post_weight / sqrt(mean(t^2) + eps)   (mean over a group)
    gate after:   t *= act(gate)
    r = residual + scale * t
    pre_weight:   h = r * pre_weight / sqrt(mean(r^2) + eps)

Every part but x is optional: the norm before a first block (pre_weight alone),
a gated norm over groups (gate_first, post_weight), or everything between two
blocks.  Device tensors run sf_block_norm; host tensors the torch form below
(the checker too).  Sums are float32 and h comes from the float32 r.  Inference
only: nothing is recorded for a backward pass."""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _lib
from ._sequences import Plans, check_apart, check_input, check_out, check_param, last_contiguous, signature

_plans = Plans()

MAX_DIM = 16384


def _rows(t: torch.Tensor, shape: Tuple[int, ...]) -> Tuple[torch.Tensor, ...]:
    """A tensor broadcast to `shape`, as up to three axes that the kernel reads in
    place: a copy where its strides allow no such view."""
    if t.shape != shape:
        t = t.expand(shape)
    t = last_contiguous(t)
    return (t.flatten(0, -3) if t.dim() > 3 else t,)


@torch.no_grad()
def _host(x, gate, act, gate_first, post_weight, group, residual, scale, pre_weight, eps):
    def norm(t, w, size):
        g = t.unflatten(-1, (-1, size))
        return (g / torch.sqrt((g * g).mean(-1, keepdim=True) + eps)).flatten(-2) * w

    t = x.float()
    if gate is not None:
        gate = gate.float()
        s = 1 / (1 + torch.exp(-gate))
        gate = gate * s if act == "silu" else s if act == "sigmoid" else gate
    if gate is not None and gate_first:
        t = t * gate
    if post_weight is not None:
        t = norm(t, post_weight, group)
    if gate is not None and not gate_first:
        t = t * gate
    if scale is not None:
        t = t * scale
    if residual is not None:
        t = residual.float() + t
    return t, None if pre_weight is None else norm(t, pre_weight, t.shape[-1])


def block_norm_forward(x: torch.Tensor, gate: Optional[torch.Tensor] = None, activation: Optional[str] = "silu",
                       gate_first: bool = False, post_weight: Optional[torch.Tensor] = None,
                       group_size: Optional[int] = None, residual: Optional[torch.Tensor] = None,
                       scale: Union[None, float, torch.Tensor] = None, pre_weight: Optional[torch.Tensor] = None,
                       eps: float = 1e-6, out: Optional[torch.Tensor] = None,
                       residual_out: Optional[torch.Tensor] = None
                       ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """x [..., dim <= 16384] -> (r, h); h is None without pre_weight.

    gate in x's type and residual in x's type or float32 broadcast to x's shape;
    post_weight, pre_weight float32 [dim]; scale a number or float32 [dim];
    group_size (of the first norm) divides dim; activation of the gate "silu",
    "sigmoid" or None.  r has the residual's type (without one, x's).  out (h)
    and residual_out (r) may be given, and each may be one of x, gate and residual;
    else they share no memory with those, nor with each other.
    """
    scale_weight = scale if isinstance(scale, torch.Tensor) else None
    factor = 1.0 if scale is None or scale_weight is not None else float(scale)
    eps, gate_first = float(eps), bool(gate_first)
    if group_size is not None:
        group_size = int(group_size)
    key = (signature(x, gate, post_weight, residual, scale_weight, pre_weight, out, residual_out), activation, gate_first,
           group_size, factor, eps)
    plan = _plans.get(key) or _plans.make(key, _check, x, gate, activation, gate_first, post_weight, group_size, residual,
                                          scale_weight, factor, pre_weight, eps, out, residual_out)
    group, r_type, desc = plan
    if out is not None or residual_out is not None:
        inputs = {"x": x, "gate": gate, "residual": residual}
        if out is not None:
            check_apart(out, "out", {**inputs, "residual_out": residual_out}, same=tuple(inputs))
        if residual_out is not None:
            check_apart(residual_out, "residual_out", inputs, same=tuple(inputs))
    if not x.is_cuda:
        r, h = _host(x, gate, activation, gate_first, post_weight, group, residual, scale, pre_weight, eps)
        r = r.to(r_type, copy=r is x) if residual_out is None else residual_out.copy_(r)
        if h is not None:
            h = h.to(x.dtype) if out is None else out.copy_(h)
        return r, h
    shape = x.shape
    if desc is None:
        # An input that the kernel does not read in place, or one to broadcast.
        x, gate, residual = (None if t is None else _rows(t, shape)[0] for t in (x, gate, residual))
        r, h = block_norm_forward(x, gate, activation, gate_first, post_weight, group_size, residual, scale, pre_weight, eps,
                                  None if out is None else out.view(x.shape),
                                  None if residual_out is None else residual_out.view(x.shape))
        return (r.view(shape) if residual_out is None else residual_out,
                None if h is None else h.view(shape) if out is None else out)
    r = torch.empty(shape, dtype=r_type, device=x.device) if residual_out is None else residual_out
    h = None
    if pre_weight is not None:
        h = torch.empty(shape, dtype=x.dtype, device=x.device) if out is None else out
    _lib.block_norm(desc, x, gate, post_weight, residual, scale_weight, pre_weight, r, h)
    return r, h


def _in_place(t: Optional[torch.Tensor], shape: torch.Size) -> Optional[Tuple[int, int]]:
    """The (outer, inner) strides of a tensor of up to three axes that the kernel
    reads in place."""
    if t is None:
        return 0, 0
    if t.shape != shape or t.dim() > 3 or (t.stride(-1) != 1 and t.shape[-1] != 1):
        return None
    return (0, 0) if t.dim() == 1 else (0, t.stride(0)) if t.dim() == 2 else (t.stride(0), t.stride(1))


def _check(x, gate, activation, gate_first, post_weight, group_size, residual, scale_weight, factor, pre_weight, eps, out,
           residual_out):
    """-> (group size, the type of r, the descriptor of a device call or None where
    an input has to be laid out first)."""
    check_input(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x is {tuple(x.shape)}: (..., dim) is wanted")
    dim, shape = int(x.shape[-1]), x.shape
    if activation not in _lib.SF_ACT:
        raise ValueError(f"activation is {activation!r}: 'silu', 'sigmoid' or None is wanted")
    if gate is not None and (gate.dtype != x.dtype or gate.device != x.device):
        raise ValueError(f"gate is {gate.dtype} on {gate.device}: {x.dtype} on {x.device} is wanted")
    if residual is not None and (residual.dtype not in (x.dtype, torch.float32) or residual.device != x.device):
        raise ValueError(f"residual is {residual.dtype} on {residual.device}: {x.dtype} or float32 on {x.device} is "
                         "wanted")
    for t, name in ((gate, "gate"), (residual, "residual")):
        if t is not None and (t.dim() > x.dim() or any(n not in (1, m) for n, m in zip(t.shape[::-1], shape[::-1]))):
            raise ValueError(f"{name} is {tuple(t.shape)}: it does not broadcast to {tuple(shape)}")
    check_param(post_weight, x, "post_weight", (dim,))
    check_param(pre_weight, x, "pre_weight", (dim,))
    check_param(scale_weight, x, "scale", (dim,))
    group = dim if group_size is None else group_size
    if group < 1 or dim % group != 0:
        raise ValueError(f"group_size {group} does not divide {dim}")
    r_type = x.dtype if residual is None else residual.dtype
    for t, name, dtype in ((out, "out", x.dtype), (residual_out, "residual_out", r_type)):
        if t is not None and (t.shape != shape or t.dtype != dtype or t.device != x.device):
            raise ValueError(f"{name} is {tuple(t.shape)} {t.dtype} on {t.device}: {tuple(shape)} {dtype} on "
                             f"{x.device} is wanted")
        check_out(t, name)
        if t is not None and x.is_cuda and (_in_place(t, shape) is None if t.dim() <= 3 else not t.is_contiguous()):
            raise ValueError(f"{name}: a contiguous last axis is wanted (over more than three axes: all of them)")
    if out is not None and pre_weight is None:
        raise ValueError("out without pre_weight: there is no second norm to write")
    if dim > MAX_DIM:
        raise _lib.UnsupportedError(f"dim {dim} is over {MAX_DIM}")
    strides = [_in_place(t, shape) for t in (x, gate, residual)]
    if not x.is_cuda or None in strides:
        return group, r_type, None
    # (New outputs have the default strides.)
    plain = _in_place(torch.empty(shape, device="meta"), shape)
    outputs = [plain if t is None else _in_place(t, shape) for t in (residual_out, out)]
    inner = 1 if x.dim() == 1 else int(shape[-2])
    outer = int(shape[0]) if x.dim() == 3 else 1
    return group, r_type, _lib.norm_desc(outer, inner, *strides, *outputs, dim, group, x.dtype, r_type, activation,
                                         bool(gate_first), float(eps), factor)
