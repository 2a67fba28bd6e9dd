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

from typing import Optional, Tuple

import torch

from .._lib import C
from .gemm import err_ptr, workspace

BLOCK = 32
NEEDS_WORKSPACE = C.NEEDS_WORKSPACE
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


def operand(t: torch.Tensor, what: str, device: int):
    """A bf16 operand of the tensor cores as ``(matrix, address, elements between rows, copy)``: rows on 16-byte boundaries. Rows that
    are not, or that are all the same one, are copied once, into rows padded to 8 elements (what a bulk-tensor load asks for); the
    address is the copy's then, which the caller holds until its launch."""
    if t.dtype is not torch.bfloat16 or t.get_device() != device:
        raise ValueError(f"{what}: expected bf16 on cuda:{device}, got {t.dtype} on {t.device}")
    t = rows2d(t, what)
    rows, cols = t.shape
    at = t.data_ptr()
    if at % 16 == 0:
        ld = t.stride(0)
        if rows <= 1:
            return t, at, -(-cols // 8) * 8, None   # one row has no stride to speak of, but a tensor map wants a multiple of 16 bytes
        if ld % 8 == 0 and ld > 0:
            return t, at, ld, None
    ld = -(-cols // 8) * 8
    padded = t.new_empty((rows, ld))
    to = padded.data_ptr()
    check(C.pad_rows(at, t.stride(0), to, ld, rows, cols, _raw_stream(device)), what)
    return t, to, ld, padded


def result(like: torch.Tensor, rows: int, cols: int) -> Tuple[torch.Tensor, int]:
    """An empty bf16 matrix and the elements between its rows: rows start on 16-byte boundaries, so that the tensor cores' next
    operator takes it as it is (``cols`` that are no multiple of 8 give a view of padded rows)."""
    if cols % 8 == 0:
        return like.new_empty((rows, cols)), cols
    ld = -(-cols // 8) * 8
    return like.new_empty((rows, ld)).narrow(1, 0, cols), ld


def vector(t: torch.Tensor, n: int, dtypes, device: int, what: str) -> int:
    """The address of ``n`` contiguous values of one of ``dtypes`` on the device."""
    if t.dim() != 1 or t.numel() != n or t.dtype not in dtypes or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{what} must be {n} contiguous values ({' or '.join(str(d) for d in dtypes)}) on cuda:{device}, "
                         f"got {tuple(t.shape)} of {t.dtype} on {t.device}")
    return t.data_ptr()


class Act8:
    """A checkpoint of ``rows x cols`` values: ``q`` int8 and ``e`` uint8, one exponent per 32 columns.

    Both are matrices with rows on 16-byte boundaries; columns past ``cols`` are padding that nothing reads. One that an operator
    makes is a single allocation, of which ``q`` and ``e`` are views that are made when asked for."""

    __slots__ = ("_q", "_e", "_both", "rows", "cols", "device_index", "_args")

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
        self._q, self._e, self._both, self.rows, self.cols = q, e, None, q.shape[0], cols
        self.device_index = q.get_device()
        self._args = (q.data_ptr(), row_stride(q), e.data_ptr(), row_stride(e))

    @classmethod
    def empty(cls, rows: int, cols: int, device) -> "Act8":
        return cls.for_rows(torch.empty((rows, 0), dtype=torch.uint8, device=device), cols)

    @classmethod
    def for_rows(cls, x: torch.Tensor, cols: int) -> "Act8":
        """An empty checkpoint for as many rows as the matrix ``x`` has, where it lives."""
        self = cls.__new__(cls)
        rows = x.shape[0]
        ldq, lde = -(-cols // 16) * 16, -(-cols // 512) * 16   # one byte of e per 32 columns; both padded to 16
        self._q = self._e = None
        self._both = both = x.new_empty(rows * (ldq + lde), dtype=torch.uint8)
        at = both.data_ptr()
        self.rows, self.cols, self.device_index, self._args = rows, cols, both.get_device(), (at, ldq, at + rows * ldq, lde)
        return self

    @property
    def q(self) -> torch.Tensor:
        if self._q is None:
            ldq = self._args[1]
            self._q = self._both[:self.rows * ldq].view(torch.int8).view(self.rows, ldq)
        return self._q

    @property
    def e(self) -> torch.Tensor:
        if self._e is None:
            self._e = self._both[self.rows * self._args[1]:].view(self.rows, self._args[3])
        return self._e

    @property
    def shape(self):
        return torch.Size((self.rows, self.cols))

    @property
    def device(self):
        return (self._q if self._both is None else self._both).device

    @property
    def nbytes(self) -> int:
        return self._q.numel() + self._e.numel() if self._both is None else self._both.numel()

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
    held = a.q if a._both is None else a._both
    s = launch_stream(held)
    x = held.new_empty((a.rows, a.cols), dtype=dtype)
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
    s, dev = launch_stream(dy), dy.get_device()
    dy2, dyp, lddy, _held = operand(dy, "act8_wgrad dy", dev)
    tokens, n = dy2.shape
    k = x8.cols
    if x8.rows != tokens or x8.device_index != dev:
        raise ValueError(f"{what}: checkpoint of {x8.rows} rows on {x8.device}, dy of {tokens} on {dy.device}")
    wp = 0 if weight is None else vector(weight, k, (torch.bfloat16,), dev, "act8_wgrad: weight")
    bp = 0 if bias is None else vector(bias, k, (torch.bfloat16,), dev, "act8_wgrad: bias")
    if bias is not None and dy_sum is None:
        raise ValueError(f"{what}: bias needs dy_sum, the sum of dy's rows")
    sp = 0 if dy_sum is None else vector(dy_sum, n, (torch.float32,), dev, "act8_wgrad: dy_sum")
    if out is None:
        if accumulate:
            raise ValueError(f"{what}: accumulate needs out")
        out = dy2.new_empty((n, k), dtype=torch.float32)
    elif out.shape != (n, k) or out.dtype is not torch.float32 or out.get_device() != dev or (k > 1 and out.stride(1) != 1):
        raise ValueError(f"{what}: out must be a {n} x {k} fp32 matrix on {dy.device} with contiguous rows")
    if tokens == 0:
        return out if accumulate else out.zero_()
    if n and k:
        need = C.act8_wgrad_scratch(tokens, n, k)
        scratch = dy2.new_empty(need, dtype=torch.uint8) if need else None
        head = (dyp, lddy, *x8._args, out.data_ptr(), row_stride(out), accumulate, wp, bp, sp, tokens, n, k, 0 if scratch is None else scratch.data_ptr())
        rc = C.act8_wgrad(*head, 0, err_ptr(dev), wait_limit_s, s)
        if rc == NEEDS_WORKSPACE:   # only where tiles are cut along the contraction
            joined = workspace(dev, s)
            rc = C.act8_wgrad(*head, joined.data_ptr(), err_ptr(dev), wait_limit_s, s)
        check(rc, what)
    return out
