"""Dropout with a mask that is never stored (``csrc/kernels/dropout.cu``).

Whether a value is kept is a function of its row, its column, a seed and an offset: the backward pass forms the same mask again, and so
does another call on rows that lie in memory in another way. The words are Philox4x32-10's (Salmon, Moraes, Dror, Shaw: "Parallel random
numbers: as easy as 1, 2, 3", SC 2011) for counter ``(column // 4, row, offset low, offset high)`` and key ``(seed low, seed high)``, 32 bits
each; a value is kept where word ``column % 4`` is at least ``round(p 2^32)``, and multiplied by ``2^32 / (2^32 - round(p 2^32))``. Rows
are counted over the leading dimensions together. Calls of one step differ in their offset.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from .._lib import C
from .act8 import _DTYPES, check, launch_stream, row_stride, rows2d

Seed = Union[int, torch.Tensor]
NO_DROPOUT = (0, 0, 0, 0, 1.0)


def drop_args(p: float, seed: Seed, offset: int, device: int, what: str):
    """``(seed, address of a seed on the device, offset, threshold, scale)`` as the native entry points take them."""
    if not 0.0 <= p < 1.0:
        raise ValueError(f"{what}: p is at least 0 and below 1, not {p!r}")
    threshold = int(p * 2.0 ** 32 + 0.5)
    if threshold >> 32:
        raise ValueError(f"{what}: p = {p!r} rounds to 1")
    at = 0
    if isinstance(seed, torch.Tensor):
        if seed.dtype is not torch.int64 or seed.numel() != 1 or seed.get_device() != device:
            raise ValueError(f"{what}: a seed in memory is one int64 on cuda:{device}, got {tuple(seed.shape)} of {seed.dtype} on {seed.device}")
        seed, at = 0, seed.data_ptr()
    elif not -(1 << 63) <= seed < 1 << 64:
        raise ValueError(f"{what}: the seed has 64 bits, {seed} has more")
    if not 0 <= offset < 1 << 64:
        raise ValueError(f"{what}: the offset is a number of 64 bits, not {offset}")
    return seed & 0xFFFFFFFFFFFFFFFF, at, offset, threshold, 2.0 ** 32 / (2 ** 32 - threshold)


def _dropout(x, p, seed, offset, residual, out, what):
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise ValueError(f"{what}: bf16 or fp32, not {x.dtype}")
    s, dev = launch_stream(x), x.get_device()
    drop = drop_args(p, seed, offset, dev, what)
    x2 = rows2d(x, what)
    rows, cols = x2.shape
    rp = ldr = 0
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.get_device() != dev:
            raise ValueError(f"{what}: residual must be like x ({tuple(x.shape)} of {x.dtype} on {x.device})")
        residual = rows2d(residual, what)
        rp, ldr = residual.data_ptr(), row_stride(residual)
    if out is None:
        y = torch.empty_like(x2) if x2.is_contiguous() else x2.new_empty((rows, cols))
    else:
        if out.shape != x.shape or out.dtype != x.dtype or out.get_device() != dev:
            raise ValueError(f"{what}: out must be like x ({tuple(x.shape)} of {x.dtype} on {x.device})")
        y = out if out.dim() == 2 else out.view(rows, cols)
        if cols > 1 and y.stride(1) != 1:
            raise ValueError(f"{what}: the values of a row of out must be contiguous")
    if rows > 0xFFFFFFFF:
        raise ValueError(f"{what}: at most 2^32 - 1 rows")
    if rows and cols:
        check(C.dropout(dt, x2.data_ptr(), row_stride(x2), rp, ldr, y.data_ptr(), row_stride(y), rows, cols, drop, s), what)
    if out is not None:
        return out
    return y if x.dim() == 2 else y.view(x.shape)


def dropout(x: torch.Tensor, p: float, seed: Seed, offset: int = 0, *, residual: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual`` + ``x`` with every value dropped with probability ``p`` (0 <= p < 1) and the others grown to match. bf16 or fp32.

    ``seed``: 64 bits, or one int64 on the device, which is read when the kernel runs (a graph that is replayed draws anew where the
    program changes it). ``offset``: another number for every call that shares a seed. What is dropped counts as 0, infinities and NaN too.
    ``out`` may be ``x`` or ``residual`` itself, and must not overlap them otherwise."""
    return _dropout(x, p, seed, offset, residual, out, "dropout")


def dropout_backward(dy: torch.Tensor, p: float, seed: Seed, offset: int = 0, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient that reaches ``x`` of :func:`dropout` with the same ``p``, ``seed`` and ``offset`` (the residual's is ``dy``)."""
    return _dropout(dy, p, seed, offset, None, out, "dropout_backward")
