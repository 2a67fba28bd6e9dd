"""Dropout with a mask that is never stored (``csrc/kernels/dropout.cu``).

Whether a value is kept is a function of its row, its column, a seed and an offset: the backward pass forms the same mask again, and so
does another call on rows that lie in memory in another way. The words are Philox4x32-10's (Salmon, Moraes, Dror, Shaw: "Parallel random
numbers: as easy as 1, 2, 3", SC 2011) for counter ``(column // 4, row, offset low, offset high)`` and key ``(seed low, seed high)``, 32 bits
each; a value is kept where word ``column % 4`` is at least ``round(p 2^32)``, and multiplied by ``2^32 / (2^32 - round(p 2^32))``. Rows
are counted over the leading dimensions together. Calls of one step differ in their offset.
"""
from __future__ import annotations

from operator import index
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
    threshold = int(p * 4294967296.0 + 0.5)
    if threshold == 4294967296:
        raise ValueError(f"{what}: p = {p!r} rounds to 1")
    at = 0
    if isinstance(seed, torch.Tensor):
        if seed.dtype is not torch.int64 or seed.numel() != 1 or seed.get_device() != device:
            raise ValueError(f"{what}: a seed in memory is one int64 on cuda:{device}, got {tuple(seed.shape)} of {seed.dtype} on {seed.device}")
        seed, at = 0, seed.data_ptr()
    else:
        seed = index(seed)
        if not -0x8000000000000000 <= seed <= 0xFFFFFFFFFFFFFFFF:
            raise ValueError(f"{what}: the seed has 64 bits, {seed} has more")
    offset = index(offset)
    if not 0 <= offset <= 0xFFFFFFFFFFFFFFFF:
        raise ValueError(f"{what}: the offset is a number of 64 bits, not {offset}")
    return seed & 0xFFFFFFFFFFFFFFFF, at, offset, threshold, 4294967296.0 / (4294967296 - threshold)


def _like_x(t, x, what, name):
    if t.shape != x.shape or t.dtype is not x.dtype or t.get_device() != x.get_device():
        raise ValueError(f"{what}: {name} must be like x ({tuple(x.shape)} of {x.dtype} on {x.device}), got {tuple(t.shape)} of {t.dtype} on {t.device}")


def _dropout(x, p, seed, offset, residual, out, what):
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise ValueError(f"{what}: bf16 or fp32, not {x.dtype}")
    s = launch_stream(x)
    drop = drop_args(p, seed, offset, x.get_device(), what)
    x2, shape = x, x.shape
    strides = x.stride()
    if len(strides) != 2 or strides[1] != 1:
        x2 = rows2d(x, what)
        strides = x2.stride()
    rows, cols = x2.shape
    ldx, rp, ldr = strides[0] if rows > 1 else cols, 0, 0
    if residual is not None:
        if residual.shape != shape or residual.dtype is not x.dtype or residual.get_device() != x.get_device():
            _like_x(residual, x, what, "residual")
        rs = residual.stride()
        if len(rs) != 2 or rs[1] != 1:
            residual = rows2d(residual, what)
            rs = residual.stride()
        rp, ldr = residual.data_ptr(), rs[0] if rows > 1 else cols
    if out is None:
        y, ldy = torch.empty_like(x2) if x2.is_contiguous() else torch.empty_strided((rows, cols), (cols, 1), dtype=x2.dtype, device=x2.device), cols
    else:
        _like_x(out, x, what, "out")
        y = out if out.dim() == 2 else out.view(rows, cols)
        if cols > 1 and y.stride(1) != 1:
            raise ValueError(f"{what}: the values of a row of out must be contiguous")
        ldy = row_stride(y)
        if rows > 1 and ldy < cols:
            raise ValueError(f"{what}: rows of out lie on one another")
    if rows > 0xFFFFFFFF:
        raise ValueError(f"{what}: at most 2^32 - 1 rows")
    if rows and cols:
        rc = C.dropout(dt, x2.data_ptr(), ldx, rp, ldr, y.data_ptr(), ldy, rows, cols, drop, s)
        if rc != 0:
            check(rc, what)
    if out is not None:
        return out
    return y if len(shape) == 2 else y.view(shape)


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
