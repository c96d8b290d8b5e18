"""Microscaled 4-bit numbers, and the Linear over weights in that format.

A row is blocks of 32 values (the last one padded with zeros): a scale byte 127 + e,
for 2^e (255: every value is NaN), and 32 codes of 4 bits, a sign and an index into
{0, .5, 1, 1.5, 2, 3, 4, 6}.  Codes are uint8 [..., 16 blocks], two to a byte with the
first in the low half, scales uint8 [..., blocks].  Quantising a block with the largest
magnitude a takes e = floor(log2 a) - 2 (at least -127) and rounds x 2^-e to the nearest
value, halfway to the even code, past 6 to 6; a block with an infinity or NaN becomes NaN.
Spikes (0 and 1) are exact.

Device tensors run sf_mx4_quantize / sf_mx4_dequantize / sf_mx4_linear; host tensors the
torch forms below.  Inference only: nothing is recorded for a backward
pass."""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _lib
from ._sequences import FLOATS, Plans, check_apart, check_input, check_out, check_param, last_contiguous, signature

Quantized = Tuple[torch.Tensor, torch.Tensor]

BLOCK = 32
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

_rows_plans, _back_plans, _linear_plans = Plans(), Plans(), Plans()


def blocks_of(size: int) -> int:
    return -(-size // BLOCK)


def _power(byte: torch.Tensor) -> torch.Tensor:
    """2^(byte - 127) in float32, from its bits."""
    byte = byte.to(torch.int32)
    return torch.where(byte > 0, byte << 23, torch.full_like(byte, 1 << 22)).view(torch.float32)


@torch.no_grad()
def host_quantize(x: torch.Tensor) -> Quantized:
    x = x.float()
    pad = -x.shape[-1] % BLOCK
    b = torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (-1, BLOCK))
    field = (b.abs().amax(-1) if b.numel() else b.sum(-1)).view(torch.int32) >> 23
    field = torch.where(torch.isnan(b).any(-1), torch.full_like(field, 255), field & 255)
    scales = torch.clamp(field - 2, min=0)
    v = b.abs() * _power(254 - scales)[..., None]
    codes = torch.zeros(v.shape, dtype=torch.uint8, device=x.device)
    for i, edge in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):  # ties go to the even code
        codes += v > edge if i % 2 == 0 else v >= edge
    codes += torch.signbit(b).to(torch.uint8) * 8
    codes[field == 255] = 0
    scales = torch.where(field == 255, torch.full_like(field, 255), scales).to(torch.uint8)
    codes = codes.flatten(-2)
    return codes[..., 0::2] + codes[..., 1::2] * 16, scales


@torch.no_grad()
def host_dequantize(codes: torch.Tensor, scales: torch.Tensor, size: int) -> torch.Tensor:
    """The first `size` values of every row, float32."""
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    pair = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    factor = _power(scales)
    factor[scales == 255] = float("nan")
    return (levels[pair.int()].unflatten(-1, (-1, BLOCK)) * factor[..., None]).flatten(-2)[..., :size]


def _pair(t, name: str) -> Quantized:
    if not isinstance(t, (tuple, list)) or len(t) != 2 or not all([isinstance(v, torch.Tensor) for v in t]):
        raise ValueError(f"{name}: a pair (codes, scales) is wanted")
    return tuple(t)


def check_quantized(t, name: str, device: torch.device) -> Quantized:
    codes, scales = _pair(t, name)
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() < 1 or codes.dim() != scales.dim() \
            or codes.shape[:-1] != scales.shape[:-1] or codes.shape[-1] != 16 * scales.shape[-1] or scales.shape[-1] < 1:
        raise ValueError(f"{name} is {tuple(codes.shape)} {codes.dtype} and {tuple(scales.shape)} {scales.dtype}: uint8 "
                         "(..., 16 blocks) and (..., blocks) are wanted")
    if codes.device != device or scales.device != device or not codes.is_contiguous() or not scales.is_contiguous():
        raise ValueError(f"{name} on {codes.device} and {scales.device}: contiguous tensors on {device} are wanted")
    return codes, scales


def _check_aligned(codes: torch.Tensor, name: str) -> None:
    """(At every call: plans know nothing of addresses.)"""
    if codes.data_ptr() % 16 != 0:
        raise ValueError(f"{name}: codes that begin at a multiple of 16 bytes are wanted")


def _rows(x: torch.Tensor) -> Optional[Tuple[int, int, Tuple[int, int]]]:
    """(outer, inner, strides) of a tensor's rows as two axes, or None where it takes more."""
    axes = [(n, s) for n, s in zip(x.shape[:-1], x.stride()[:-1]) if n != 1]
    merged = []
    for n, s in axes:
        if merged and merged[-1][1] == n * s:
            merged[-1] = (merged[-1][0] * n, s)
        else:
            merged.append((n, s))
    if len(merged) > 2:
        return None
    merged = [(1, 0)] * (2 - len(merged)) + merged
    return merged[0][0], merged[1][0], (merged[0][1], merged[1][1])


def mx4_quantize(x: torch.Tensor, out: Optional[Quantized] = None) -> Quantized:
    """x [..., dim] -> (codes [..., 16 blocks], scales [..., blocks]); out: such a pair to write."""
    if x.is_cuda and x.dim() > 0:
        x = last_contiguous(x)
    if out is not None:
        out = _pair(out, "out")
    key = (signature(x), None if out is None else signature(*out))
    rows, shapes = _rows_plans.get(key) or _rows_plans.make(key, _check_quantize, x, out)
    if out is None:
        out = (torch.empty(shapes[0], dtype=torch.uint8, device=x.device), torch.empty(shapes[1], dtype=torch.uint8, device=x.device))
    else:
        if x.is_cuda:
            _check_aligned(out[0], "out")
        check_apart(out[0], "out's codes", {"x": x, "out's scales": out[1]})
        check_apart(out[1], "out's scales", {"x": x})
    if not x.is_cuda:
        for t, v in zip(out, host_quantize(x)):
            t.copy_(v)
        return out
    if rows is None:
        x = x.contiguous()
        rows = _rows(x)
    _lib.mx4_quantize(x, *rows, *out)
    return out


def _check_quantize(x, out):
    check_input(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x is {tuple(x.shape)}: (..., dim) is wanted")
    n = blocks_of(int(x.shape[-1]))
    shapes = (x.shape[:-1] + (16 * n,), x.shape[:-1] + (n,))
    if out is not None:
        codes, scales = check_quantized(out, "out", x.device)
        if codes.shape != shapes[0]:
            raise ValueError(f"out is {tuple(codes.shape)} and {tuple(scales.shape)}: {tuple(shapes[0])} and "
                             f"{tuple(shapes[1])} are wanted")
    return _rows(x), shapes


def mx4_dequantize(codes: torch.Tensor, scales: torch.Tensor, size: Optional[int] = None,
                   dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(codes, scales) -> [..., size] (default: whole blocks) in `dtype`, or into a contiguous out."""
    if size is not None:
        size = int(size)
    key = (signature(codes, scales, out), size, dtype)
    shape, dtype, rows = _back_plans.get(key) or _back_plans.make(key, _check_dequantize, codes, scales, size, dtype, out)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=codes.device)
    else:
        check_apart(out, "out", {"codes": codes, "scales": scales})
    if not codes.is_cuda:
        return out.copy_(host_dequantize(codes, scales, shape[-1]))
    _check_aligned(codes, "codes, scales")
    _lib.mx4_dequantize(codes, scales, rows, out)
    return out


def _check_dequantize(codes, scales, size, dtype, out):
    """-> (the result's shape and type, rows)."""
    check_quantized((codes, scales), "codes, scales", codes.device)
    n = int(scales.shape[-1])
    size = BLOCK * n if size is None else size
    if blocks_of(size) != n:
        raise ValueError(f"size {size}: rows of {n} blocks have {BLOCK * (n - 1) + 1} to {BLOCK * n} values")
    shape = codes.shape[:-1] + (size,)
    if out is not None:
        if out.shape != shape or out.dtype not in FLOATS or out.device != codes.device or not out.is_contiguous():
            raise ValueError(f"out is {tuple(out.shape)} {out.dtype} on {out.device}: a contiguous {tuple(shape)} float "
                             f"tensor on {codes.device} is wanted")
        dtype = out.dtype
    elif dtype not in FLOATS:
        raise _lib.UnsupportedError(f"dtype is {dtype}: float32, float16 or bfloat16 is wanted")
    return shape, dtype, codes.numel() // (16 * n)


def mx4_linear_forward(x: Union[torch.Tensor, Quantized], weight: Quantized, bias: Optional[torch.Tensor] = None,
                       dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [..., K] W^T + bias -> [..., N], W a quantised [N, K], bias float32 [N].

    x as floats is taken as it is (every product is exact, sums are float32; of float32 x
    the bits from 2^-133 on count, and weights past float32, of scales 253 and 254, are
    infinite or NaN); as a pair (codes, scales) of rows of as many blocks it goes to the 4-bit matrix
    instructions.  The result has `dtype` (default x's, for a pair float32) or out's;
    out shares no memory with the inputs.
    """
    four = not isinstance(x, torch.Tensor)
    x_scales = None
    if four:
        x, x_scales = _pair(x, "x")
    w, w_scales = weight = _pair(weight, "weight")
    key = (signature(x, x_scales, *weight, bias, out), dtype)
    plan = _linear_plans.get(key) or _linear_plans.make(key, _check_linear, x, x_scales, weight, bias, dtype, out)
    shape, dtype, desc, flat = plan
    if x.is_cuda:
        _check_aligned(w, "weight")
        if four:
            _check_aligned(x, "x")
    if out is None:
        y = torch.empty(shape, dtype=dtype, device=x.device)
    else:
        y = out
        check_apart(out, "out", {"x": x, "x's scales": x_scales, "weight": w, "weight's scales": w_scales, "bias": bias})
    if not x.is_cuda:
        k = BLOCK * w_scales.shape[-1] if four else x.shape[-1]
        with torch.no_grad():
            r = (host_dequantize(x, x_scales, k) if four else x.float()) @ host_dequantize(w, w_scales, k).t()
            return y.copy_(r if bias is None else r + bias)
    if desc is None:
        x = x.contiguous()
        desc = _lib.mx4_linear_desc(flat[0], w.shape[0], x.shape[-1], x.shape[-1], flat[1], x.dtype, dtype)
    _lib.mx4_linear(desc, x, x_scales, w, w_scales, bias, y)
    return y


def _check_linear(x, x_scales, weight, bias, dtype, out):
    """-> (y's shape and type, the descriptor of a device call or None where x has to be
    laid out first, (rows, y's row stride))."""
    if x_scales is not None:
        check_quantized((x, x_scales), "x", x.device)
    w, w_scales = check_quantized(weight, "weight", x.device)
    if w.dim() != 2 or w.shape[0] < 1:
        raise ValueError(f"weight is {tuple(w.shape)}: (N, 16 blocks) is wanted")
    n = int(w.shape[0])
    if x_scales is None:
        check_input(x, "x")
        if x.dim() < 1 or x.shape[-1] < 1 or blocks_of(int(x.shape[-1])) != w_scales.shape[1]:
            raise ValueError(f"x is {tuple(x.shape)}: (..., K) of the weight's {w_scales.shape[1]} blocks is wanted")
        k = int(x.shape[-1])
    else:
        if x_scales.shape[-1] != w_scales.shape[1]:
            raise ValueError(f"x has {x_scales.shape[-1]} blocks: the weight's {w_scales.shape[1]} are wanted")
        k = BLOCK * int(x_scales.shape[-1])
    check_param(bias, x, "bias", (n,))
    shape = x.shape[:-1] + (n,)
    if out is not None:
        if dtype is not None and dtype != out.dtype:
            raise ValueError(f"out is {out.dtype}: {dtype} is wanted")
        dtype = out.dtype
        if out.shape != shape or out.device != x.device:
            raise ValueError(f"out is {tuple(out.shape)} on {out.device}: {tuple(shape)} on {x.device} is wanted")
        check_out(out, "out")
    dtype = dtype or (torch.float32 if x_scales is not None else x.dtype)
    if dtype not in FLOATS:
        raise _lib.UnsupportedError(f"dtype is {dtype}: float32, float16 or bfloat16 is wanted")
    rows = 1
    for v in x.shape[:-1]:
        rows *= int(v)
    ys = n
    if out is not None:
        at = _rows(out)
        if (out.stride(-1) != 1 and n > 1) or at is None or at[0] != 1:
            raise ValueError("out: rows at one stride with a contiguous last axis are wanted")
        ys = at[2][1]
    if not x.is_cuda:
        return shape, dtype, None, (rows, ys)
    if x_scales is not None:
        return shape, dtype, _lib.mx4_linear_desc(rows, n, k, 0, ys, None, dtype), (rows, ys)
    at = _rows(x)
    if (x.stride(-1) != 1 and k > 1) or at is None or at[0] != 1:
        return shape, dtype, None, (rows, ys)
    return shape, dtype, _lib.mx4_linear_desc(rows, n, k, at[2][1], ys, x.dtype, dtype), (rows, ys)
