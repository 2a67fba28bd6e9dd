"""Activation checkpoints in 8 bits: what the backward pass needs of the forward pass in half the memory of bf16.

32 neighbours of a row share a power of two: ``x`` is kept as whole numbers ``q`` of -127..127 and a step ``2^(e-127)``, the
smallest at which the largest of the 32 rounds to at most 127, so a value is off by half a step at most (under 1/127 of the
largest of its block). A block that held an infinity or NaN comes back as NaN. Values ``q * 2^(e-127)`` are exact in bf16.

``act8_pack`` / ``act8_unpack`` convert rows (``csrc/kernels/norm.cu``). ``norm.layer_norm_act8`` and ``linear.linear_act``
write a checkpoint beside their output, and the backward passes read it as it is: ``norm.layer_norm_act8_backward``,
``linear.linear_act_dgrad`` and ``act8_wgrad``, the weight gradient with a checkpoint as one operand
(``csrc/kernels/act8_wgrad.cu``).
"""
from __future__ import annotations

from typing import Optional

import torch

from .._lib import C

BLOCK = 32
_DTYPES = {torch.bfloat16: 0, torch.float32: 1}


def launch_stream(t: torch.Tensor) -> int:
    """The current stream's handle; refuses a tensor that lives on another device than the current one."""
    if not t.is_cuda:
        raise ValueError(f"expected CUDA tensors, got one on {t.device}")
    s = torch.cuda.current_stream()
    if s.device_index != t.get_device():
        raise ValueError(f"tensor on cuda:{t.get_device()}, but the current device is cuda:{s.device_index}")
    return s.cuda_stream


def rows2d(t: torch.Tensor, what: str) -> torch.Tensor:
    """``t`` as a matrix of its rows (last dimension); rows may be strided, values of a row may not."""
    if t.dim() == 0:
        raise ValueError(f"{what}: needs at least one dimension")
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1]) if t.shape[-1] else t.reshape(0, 0)
    if t.stride(1) != 1 and t.shape[1] > 1:
        t = t.contiguous()
    return t


def row_stride(t: torch.Tensor) -> int:
    """Elements between rows (a matrix of one row may report any stride: it has none)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


class Act8:
    """A checkpoint of ``rows x cols`` values: ``q`` int8 and ``e`` uint8, one exponent per 32 columns.

    Both are matrices with rows on 16-byte boundaries; columns past ``cols`` are padding that nothing reads."""

    __slots__ = ("q", "e", "rows", "cols")

    def __init__(self, q: torch.Tensor, e: torch.Tensor, cols: int):
        if q.dtype != torch.int8 or e.dtype != torch.uint8 or q.dim() != 2 or e.dim() != 2 or q.shape[0] != e.shape[0]:
            raise ValueError("Act8: q is an int8 matrix, e a uint8 matrix of as many rows")
        if q.device != e.device:
            raise ValueError("Act8: q and e are on different devices")
        if cols < 0 or q.shape[1] < cols or e.shape[1] * BLOCK < cols:
            raise ValueError(f"Act8: {cols} columns do not fit q of {q.shape[1]} and e of {e.shape[1]} columns")
        if q.numel() and (q.stride(1) != 1 or e.stride(1) != 1 or row_stride(q) % 16 or row_stride(e) % 16
                          or q.data_ptr() % 16 or e.data_ptr() % 16):
            raise ValueError("Act8: rows of q and e start on 16-byte boundaries")
        self.q, self.e, self.rows, self.cols = q, e, q.shape[0], cols

    @classmethod
    def empty(cls, rows: int, cols: int, device) -> "Act8":
        ldq, lde = -(-cols // 16) * 16, -(-(-(-cols // BLOCK)) // 16) * 16
        self = cls.__new__(cls)
        self.q = torch.empty((rows, ldq), dtype=torch.int8, device=device)
        self.e = torch.empty((rows, lde), dtype=torch.uint8, device=device)
        self.rows, self.cols = rows, cols
        return self

    @property
    def shape(self):
        return torch.Size((self.rows, self.cols))

    @property
    def device(self):
        return self.q.device

    @property
    def nbytes(self) -> int:
        return self.q.numel() + self.e.numel()

    def args(self):
        """(q, ldq, e, lde) as the native entry points take them."""
        return self.q.data_ptr(), row_stride(self.q), self.e.data_ptr(), row_stride(self.e)

    def __repr__(self) -> str:
        return f"Act8({self.rows} x {self.cols}, {self.device})"


def check(rc: int, what: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{what} failed with code {rc}")


def act8_pack(x: torch.Tensor) -> Act8:
    """The 8-bit checkpoint of ``x`` (bf16 or fp32; leading dimensions are taken together as rows)."""
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise ValueError(f"act8_pack: bf16 or fp32, not {x.dtype}")
    s = launch_stream(x)
    x = rows2d(x, "act8_pack")
    out = Act8.empty(x.shape[0], x.shape[1], x.device)
    check(C.act8_pack(dt, x.data_ptr(), row_stride(x), *out.args(), out.rows, out.cols, s), "act8_pack")
    return out


def act8_unpack(a: Act8, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that a checkpoint stands for, as a ``rows x cols`` matrix (exact in either type)."""
    dt = _DTYPES.get(dtype)
    if dt is None:
        raise ValueError(f"act8_unpack: bf16 or fp32, not {dtype}")
    s = launch_stream(a.q)
    x = torch.empty((a.rows, a.cols), dtype=dtype, device=a.q.device)
    check(C.act8_unpack(dt, *a.args(), x.data_ptr(), a.cols, a.rows, a.cols, s), "act8_unpack")
    return x
