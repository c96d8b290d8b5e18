"""What the state space entry points share: their checks of arguments, and
sequences and state pools on host tensors.

A prompt comes dense, [batch, tokens, ...], or packed, [total, ...] with
`offsets` (int32 [sequences + 1]): sequence b is rows offsets[b] to
offsets[b + 1] - 1.  The state of sequence b is row slots[b] of a pool (without
slots: row b)."""

from __future__ import annotations

from typing import Callable, List, Optional, Tuple

import torch

FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def signature(*tensors: Optional[torch.Tensor]) -> tuple:
    """Everything about a call's tensors but their addresses and values."""
    return tuple([None if t is None else (t.shape, t.stride(), t.dtype, t.get_device()) for t in tensors])


class Plans(dict):
    """What a checked call with a signature comes to.  A decoding loop repeats its
    calls, and checking the tensors of one again costs as much as launching it
    (a step of the scan: 14 us with, 9 without).  The keys hold plain values: a
    number that comes as a tensor is read at every call."""

    MOST = 4096

    def make(self, key: tuple, check: Callable, *args):
        plan = check(*args)
        if len(self) >= self.MOST:
            self.clear()
        self[key] = plan
        return plan


def check_input(t: torch.Tensor, name: str) -> None:
    if t.dtype not in FLOATS:
        from .. import _lib

        raise _lib.UnsupportedError(f"{name} is {t.dtype}: float32, float16 or bfloat16 is wanted")


def check_like(t: torch.Tensor, x: torch.Tensor, name: str, shape: Tuple[int, ...]) -> None:
    if tuple(t.shape) != shape or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{name} is {tuple(t.shape)} {t.dtype} on {t.device}: {shape} {x.dtype} on {x.device} is wanted")


def check_param(t: Optional[torch.Tensor], x: torch.Tensor, name: str, shape: Tuple[int, ...]) -> None:
    if t is None:
        return
    if tuple(t.shape) != shape or t.dtype != torch.float32 or t.device != x.device or not t.is_contiguous():
        raise ValueError(f"{name} is {tuple(t.shape)} {t.dtype} on {t.device}: a contiguous {shape} float32 on "
                         f"{x.device} is wanted")


def check_index(t: Optional[torch.Tensor], x: torch.Tensor, name: str, size: int) -> None:
    if t is None:
        return
    if t.dim() != 1 or t.numel() != size or t.dtype != torch.int32 or t.device != x.device or not t.is_contiguous():
        raise ValueError(f"{name} is {tuple(t.shape)} {t.dtype} on {t.device}: a contiguous ({size},) int32 on "
                         f"{x.device} is wanted")


def check_pool(t: Optional[torch.Tensor], x: torch.Tensor, name: str, row: Tuple[int, ...], dtype: torch.dtype,
               batch: int, slots: Optional[torch.Tensor]) -> None:
    if t is None:
        return
    if t.dim() != len(row) + 1 or tuple(t.shape[1:]) != row or t.dtype != dtype or t.device != x.device \
            or not t.is_contiguous() or (slots is None and t.shape[0] != batch):
        rows = f"{batch}" if slots is None else "rows"
        raise ValueError(f"{name} is {tuple(t.shape)} {t.dtype} on {t.device}: a contiguous "
                         f"({rows}, {', '.join(map(str, row))}) {dtype} on {x.device} is wanted")


def check_out(t: Optional[torch.Tensor], name: str) -> None:
    if t is not None and any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)):
        raise ValueError(f"{name} is an expanded tensor: elements of its own are wanted")


def _reach(t: torch.Tensor) -> int:
    """Bytes from a tensor's first element to the end of its last."""
    if t.is_contiguous():
        return t.numel() * t.element_size()
    return (1 + sum([(n - 1) * s for n, s in zip(t.shape, t.stride())])) * t.element_size()


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether elements of a and b share memory.  (Views of one buffer that lie side by
    side along any of its axes do not.)"""
    by = b.data_ptr() - a.data_ptr()
    if by >= _reach(a) or -by >= _reach(b) or a.numel() == 0 or b.numel() == 0:
        return False
    # Modulo a step that all longer ones are multiples of: what the shorter ones reach.
    axes = [[(s * t.element_size(), n) for s, n in zip(t.stride(), t.shape) if n > 1] for t in (a, b)]
    for step in {s for own in axes for s, _ in own if s > 0}:
        if any(s > step and s % step for own in axes for s, _ in own):
            continue
        inner = [t.element_size() + sum([s * (n - 1) for s, n in own if s < step]) for t, own in zip((a, b), axes)]
        if by % step >= inner[0] and by % step + inner[1] <= step:
            return False
    return True


def check_apart(written: torch.Tensor, name: str, others: dict, same: Tuple[str, ...] = ()) -> None:
    """What a call writes shares no memory with what it reads; those of `same` it may be."""
    for other, t in others.items():
        if t is None or not overlap(written, t):
            continue
        if other not in same or t.data_ptr() != written.data_ptr() or t.shape != written.shape or t.dtype != written.dtype \
                or any(a != b and n > 1 for a, b, n in zip(t.stride(), written.stride(), t.shape)):
            raise ValueError(f"{name} shares memory with {other}")


def last_contiguous(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def host_spans(x: torch.Tensor, offsets: Optional[torch.Tensor]) -> List[torch.Tensor]:
    """Host: every sequence's [tokens, ...] view of x."""
    if offsets is None:
        return list(x.unbind(0))
    total = x.shape[0]
    at = [min(max(int(v), 0), total) for v in offsets]
    return [x[a:max(a, b)] for a, b in zip(at, at[1:])]


def host_slots(batch: int, rows: int, slots: Optional[torch.Tensor]) -> List[int]:
    """Host: every sequence's row of the pool, -1 where it has none."""
    pick = range(batch) if slots is None else [int(v) for v in slots]
    return [s if 0 <= s < rows else -1 for s in pick]
