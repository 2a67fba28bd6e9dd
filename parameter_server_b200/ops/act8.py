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
from .gemm import _err_flag, workspace

BLOCK = 32
_DTYPES = {torch.bfloat16: 0, torch.float32: 1}


# (``torch.cuda.current_stream()`` builds a Stream object: 3 us, as much as a small launch)
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def launch_stream(t: torch.Tensor) -> int:
    """The current stream's handle; refuses a tensor that lives on another device than the current one."""
    if not t.is_cuda:
        raise ValueError(f"expected CUDA tensors, got one on {t.device}")
    d = t.get_device()
    if d != _current_device():
        raise ValueError(f"tensor on cuda:{d}, but the current device is cuda:{_current_device()}")
    return _raw_stream(d)


def rows2d(t: torch.Tensor, what: str) -> torch.Tensor:
    """``t`` as a matrix of its rows (last dimension); rows may be strided, values of a row may not."""
    if t.dim() == 2 and t.stride(1) == 1:
        return t
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


def _matrix(t: torch.Tensor, what: str, like: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A bf16 operand of the tensor cores: rows on 16-byte boundaries. Rows that are not are copied once, into rows padded to
    8 elements (what a bulk-tensor load asks for)."""
    if t.dtype != torch.bfloat16 or (like is not None and t.get_device() != like.get_device()):
        raise ValueError(f"{what}: expected bf16" + ("" if like is None else f" on {like.device}") + f", got {t.dtype} on {t.device}")
    t = rows2d(t, what)
    if row_stride(t) % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    rows, cols = t.shape
    padded = torch.empty((rows, -(-cols // 8) * 8), dtype=t.dtype, device=t.device)[:, :cols]
    padded.copy_(t)
    return padded


def _ld(t: torch.Tensor) -> int:
    # one row has no stride to speak of, but a tensor map wants a multiple of 16 bytes
    return t.stride(0) if t.shape[0] > 1 else -(-t.shape[1] // 8) * 8


class Act8:
    """A checkpoint of ``rows x cols`` values: ``q`` int8 and ``e`` uint8, one exponent per 32 columns.

    Both are matrices with rows on 16-byte boundaries; columns past ``cols`` are padding that nothing reads."""

    __slots__ = ("q", "e", "rows", "cols", "_args")

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
        self._args = (q.data_ptr(), row_stride(q), e.data_ptr(), row_stride(e))

    @classmethod
    def empty(cls, rows: int, cols: int, device) -> "Act8":
        return cls._like(torch.empty((rows, -(-cols // 16) * 16), dtype=torch.int8, device=device), cols)

    @classmethod
    def for_rows(cls, x: torch.Tensor, cols: int) -> "Act8":
        """An empty checkpoint for as many rows as the matrix ``x`` has, where it lives."""
        return cls._like(x.new_empty((x.shape[0], -(-cols // 16) * 16), dtype=torch.int8), cols)

    @classmethod
    def _like(cls, q: torch.Tensor, cols: int) -> "Act8":
        rows, ldq = q.shape
        lde = -(-cols // 512) * 16   # one byte per 32 columns, padded to 16
        self = cls.__new__(cls)
        self.q = q
        self.e = q.new_empty((rows, lde), dtype=torch.uint8)
        self.rows, self.cols = rows, cols
        self._args = (self.q.data_ptr(), ldq, self.e.data_ptr(), lde)
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
        return self._args

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
    out = Act8.for_rows(x, x.shape[1])
    check(C.act8_pack(dt, x.data_ptr(), row_stride(x), *out.args(), out.rows, out.cols, s), "act8_pack")
    return out


def act8_unpack(a: Act8, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that a checkpoint stands for, as a ``rows x cols`` matrix (exact in either type)."""
    dt = _DTYPES.get(dtype)
    if dt is None:
        raise ValueError(f"act8_unpack: bf16 or fp32, not {dtype}")
    s = launch_stream(a.q)
    x = a.q.new_empty((a.rows, a.cols), dtype=dtype)
    check(C.act8_unpack(dt, *a.args(), x.data_ptr(), a.cols, a.rows, a.cols, s), "act8_unpack")
    return x


def act8_wgrad(dy: torch.Tensor, x8: Act8, *, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               dy_sum: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, accumulate: bool = False,
               wait_limit_s: float = 2.0) -> torch.Tensor:
    """``dy^T x`` in fp32, ``[N, K]``, for ``dy`` ``[..., N]`` (bf16) and the layer's input ``x`` (rows of ``K``) as an 8-bit checkpoint.

    ``weight`` and ``bias`` (bf16, ``[K]``): the layer's input was a layer norm's output and ``x8`` holds its normalised rows
    (``norm.layer_norm_act8``), so the operand is ``x * weight + bias``. With ``bias``, ``dy_sum`` is the sum of dy's rows (fp32, ``[N]``:
    the layer's bias gradient, ``linear.linear_bias_grad``). ``out`` is written, or added to with ``accumulate``."""
    what = "act8_wgrad"
    s = launch_stream(dy)
    dy2 = _matrix(dy, f"{what} dy")
    tokens, n = dy2.shape
    k = x8.cols
    if x8.rows != tokens or x8.device != dy.device:
        raise ValueError(f"{what}: checkpoint of {x8.rows} rows on {x8.device}, dy of {tokens} on {dy.device}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.shape != (k,) or t.dtype != torch.bfloat16 or t.device != dy.device or not t.is_contiguous()):
            raise ValueError(f"{what}: {name} must be {k} contiguous bf16 values on {dy.device}")
    if bias is not None and dy_sum is None:
        raise ValueError(f"{what}: bias needs dy_sum, the sum of dy's rows")
    if dy_sum is not None and (dy_sum.shape != (n,) or dy_sum.dtype != torch.float32 or dy_sum.device != dy.device or not dy_sum.is_contiguous()):
        raise ValueError(f"{what}: dy_sum must be {n} contiguous fp32 values on {dy.device}")
    if out is None:
        if accumulate:
            raise ValueError(f"{what}: accumulate needs out")
        out = dy2.new_empty((n, k), dtype=torch.float32)
    elif out.shape != (n, k) or out.dtype != torch.float32 or out.device != dy.device or (k > 1 and out.stride(1) != 1):
        raise ValueError(f"{what}: out must be a {n} x {k} fp32 matrix on {dy.device} with contiguous rows")
    if tokens == 0:
        return out if accumulate else out.zero_()
    if n and k:
        need = C.act8_wgrad_scratch(tokens, n, k)
        scratch = torch.empty(need, dtype=torch.uint8, device=dy.device) if need else None
        head = (dy2.data_ptr(), _ld(dy2), *x8.args(), out.data_ptr(), row_stride(out), accumulate, 0 if weight is None else weight.data_ptr(),
                0 if bias is None else bias.data_ptr(), 0 if dy_sum is None else dy_sum.data_ptr(), tokens, n, k,
                0 if scratch is None else scratch.data_ptr())
        tail = (_err_flag(dy.device).data_ptr(), wait_limit_s, s)
        rc = C.act8_wgrad(*head, 0, *tail)
        if rc == C.NEEDS_WORKSPACE:   # only where tiles are cut along the contraction
            joined = workspace(dy.get_device(), s)
            rc = C.act8_wgrad(*head, joined.data_ptr(), *tail)
        check(rc, what)
    return out
