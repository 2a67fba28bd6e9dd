"""Linear layers of a decoder block with their neighbours in the epilogue (``csrc/kernels/linear_fused.cuh``), bf16 operands and
fp32 sums:

* ``linear_act``: ``act(x w^T + b) + residual``, with the value before the activation kept for the backward pass, and dropout between;
* ``linear_act_dgrad``: the gradient that reaches that value, ``(dy w) * act'(h)``, and ``act(h)`` again;
* ``linear_bias_grad``: the sum of dy's rows in a fixed order.

The weight gradient is ``ops.gemm.linear_wgrad``, or ``ops.act8.act8_wgrad`` from an 8-bit checkpoint. A bounded wait that ran out
is reported by ``ops.gemm.check_gemm_errors``.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from .._lib import C
from .act8 import _DTYPES, NEEDS_WORKSPACE, Act8, check, launch_stream, operand, result, row_stride, rows2d, vector
from .dropout import NO_DROPOUT, drop_args
from .gemm import err_ptr, workspace

ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
_BIAS_TYPES = (torch.bfloat16, torch.float32)
_NOT_KEPT = (0, 0, 0, 0)


def _act_code(act, what: str) -> int:
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"{what}: act is one of {sorted(k for k in ACTIVATIONS if k)}, not {act!r}")
    return code


def _like(t: torch.Tensor, shape, device: int, what: str) -> None:
    if t.shape != shape or t.dtype is not torch.bfloat16 or t.get_device() != device:
        raise ValueError(f"{what} must be {tuple(shape)} bf16 on cuda:{device}, got {tuple(t.shape)} of {t.dtype} on {t.device}")


def _beside(t: torch.Tensor, what: str, device: int):
    """``(address, elements between rows, what to hold)`` of a matrix that the epilogue reads. A large one whose rows do not start on
    16-byte boundaries is padded first: 15376 x 3607, 39 us, where reading it as it lies costs 570."""
    t = rows2d(t, what)
    ld, at = row_stride(t), t.data_ptr()
    if (ld % 8 or at % 16) and t.numel() > 1 << 19:
        return operand(t, what, device)[1:]
    return at, ld, t


def _run(dev, s, what, args, limit):
    err = err_ptr(dev)
    rc = C.linear_fused(*args, 0, err, limit, s)
    if rc == NEEDS_WORKSPACE:   # only where tiles are cut along the contraction
        scratch = workspace(dev, s)
        rc = C.linear_fused(*args, scratch.data_ptr(), err, limit, s)
    if rc != 0:
        check(rc, what)


def linear_act(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, *, act: Optional[str] = None,
               residual: Optional[torch.Tensor] = None, save: Optional[str] = None, out: Optional[torch.Tensor] = None,
               dropout: Optional[tuple] = None, wait_limit_s: float = 2.0):
    """``act(x w^T + bias) + residual`` for ``x`` ``[..., K]``, ``w`` ``[N, K]`` (bf16), ``bias`` ``[N]`` (bf16 or fp32) and
    ``residual`` ``[..., N]`` (bf16). ``act``: "none", "relu", "gelu", "gelu_tanh" or "silu".

    ``save`` = "bf16" or "act8" also returns ``h = x w^T + bias`` as :func:`linear_act_dgrad` takes it: ``(y, h)`` with ``h`` a bf16
    tensor like ``y``, or an :class:`~.act8.Act8`. ``dropout`` = ``(p, seed, offset)`` drops values behind the activation, ahead of the residual,
    as :func:`~.dropout.dropout` does with the same three (``dropout_backward`` takes the gradient back). ``out`` (bf16, may be ``residual`` itself) receives ``y``. Results whose ``N`` is no
    multiple of 8 have padded rows (``stride(-2)``), as the next product wants them."""
    what = "linear_act"
    code = _act_code(act, what)
    if save not in (None, "bf16", "act8"):
        raise ValueError(f"{what}: save is None, 'bf16' or 'act8', not {save!r}")
    s, dev = launch_stream(x), x.get_device()
    drop = NO_DROPOUT
    if dropout is not None:
        if not isinstance(dropout, (tuple, list)) or len(dropout) != 3:
            raise ValueError(f"{what}: dropout is (p, seed, offset), not {dropout!r}")
        drop = drop_args(*dropout, dev, what)
    x2, xp, ldx, _held = operand(x, "linear_act x", dev)
    w, wp, ldw, _held_w = operand(w, "linear_act w", dev)
    M, K = x2.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"{what}: x has {K} columns, w has {w.shape[1]}")
    if K == 0:
        raise ValueError(f"{what}: a sum over no columns")
    bp = 0 if bias is None else vector(bias, N, _BIAS_TYPES, dev, "linear_act: bias")
    shape = None if residual is None and out is None and x.dim() == 2 else x.shape[:-1] + (N,)
    rp, ldr, _held_r = 0, 0, None
    if residual is not None:
        _like(residual, shape, dev, "linear_act: residual")
        rp, ldr, _held_r = _beside(residual, what, dev)
    if out is None:
        y, ldy = result(x2, M, N)
    else:
        _like(out, shape, dev, "linear_act: out")
        y = out if out.dim() == 2 else out.view(M, N)
        if N > 1 and y.stride(1) != 1:
            raise ValueError(f"{what}: the values of a row of out must be contiguous")
        ldy = row_stride(y)
    pre, ldpre = result(x2, M, N) if save == "bf16" else (None, 0)
    kept = Act8.for_rows(y, N) if save == "act8" else None
    if M and N:
        _run(dev, s, what, (False, False, code, M, N, K, xp, ldx, wp, ldw, bp, bias is not None and bias.dtype is torch.float32,
                            rp, ldr, y.data_ptr(), ldy, 0, 0, 0 if pre is None else pre.data_ptr(), ldpre,
                            *(_NOT_KEPT if kept is None else kept._args), 0, 0, 0, 0, drop), wait_limit_s)
    if out is not None:
        y = out
    elif x.dim() != 2:
        y = y.view(shape)
    if save is None:
        return y
    return y, (kept if pre is None else pre if x.dim() == 2 else pre.view(x.shape[:-1] + (N,)))


def linear_act_dgrad(dy: torch.Tensor, w: torch.Tensor, h: Union[torch.Tensor, Act8, None], *, act: Optional[str] = None,
                     recompute: bool = False, wait_limit_s: float = 2.0):
    """``(dy w) * act'(h)`` for ``dy`` ``[..., K]`` and the weight ``w`` ``[K, N]`` (as the forward pass has it: ``y = a w^T``) of the
    layer that took ``a = act(h)``; ``h`` ``[..., N]`` is what ``linear_act(save=...)`` returned (None where ``act`` is "none").
    With ``recompute``: ``(dh, a)``, where ``a`` (bf16) is what the weight gradient of that layer needs."""
    what = "linear_act_dgrad"
    code = _act_code(act, what)
    s, dev = launch_stream(dy), dy.get_device()
    dy2, dyp, lddy, _held = operand(dy, "linear_act_dgrad dy", dev)
    w, wp, ldw, _held_w = operand(w, "linear_act_dgrad w", dev)
    M, K = dy2.shape
    N = w.shape[1]
    if w.shape[0] != K:
        raise ValueError(f"{what}: dy has {K} columns, w has {w.shape[0]} rows")
    if K == 0:
        raise ValueError(f"{what}: a sum over no columns")
    pre, ldpre, _held_h, kept = 0, 0, None, None
    if isinstance(h, Act8):
        if h.rows != M or h.cols != N or h.device_index != dev:
            raise ValueError(f"{what}: checkpoint of {h.rows} x {h.cols} on {h.device}, expected {M} x {N} on {dy.device}")
        kept = h
    elif h is not None:
        _like(h, dy.shape[:-1] + (N,), dev, "linear_act_dgrad: h")
        pre, ldpre, _held_h = _beside(h, what, dev)
    elif code != 0 or recompute:
        raise ValueError(f"{what}: h is needed")
    dh, ld = result(dy2, M, N)
    a = result(dy2, M, N)[0] if recompute else None
    if M and N:
        _run(dev, s, what, (True, False, code, M, N, K, dyp, lddy, wp, ldw, 0, False, 0, 0, dh.data_ptr(), ld, 0 if a is None else a.data_ptr(), ld,
                            pre, ldpre, *(_NOT_KEPT if kept is None else kept._args), 0, 0, 0, 0, NO_DROPOUT), wait_limit_s)
    if dy.dim() != 2:
        shape = dy.shape[:-1] + (N,)
        dh = dh.view(shape)
        a = None if a is None else a.view(shape)
    return (dh, a) if recompute else dh


def linear_bias_grad(dy: torch.Tensor, out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """The bias gradient: the sum of dy's rows in fp32, in a fixed order. Written to ``out`` (fp32), or added to it."""
    dt = _DTYPES.get(dy.dtype)
    if dt is None:
        raise ValueError(f"linear_bias_grad: bf16 or fp32, not {dy.dtype}")
    s = launch_stream(dy)
    dy2 = rows2d(dy, "linear_bias_grad")
    rows, n = dy2.shape
    if out is None:
        if accumulate:
            raise ValueError("linear_bias_grad: accumulate needs out")
        out = dy2.new_empty(n, dtype=torch.float32)
    elif out.dtype != torch.float32 or out.shape != (n,) or out.device != dy.device or not out.is_contiguous():
        raise ValueError(f"linear_bias_grad: out must be {n} contiguous fp32 values on {dy.device}")
    partial = dy2.new_empty(C.column_sum_scratch(rows, n), dtype=torch.float32)
    check(C.column_sum(dt, dy2.data_ptr(), row_stride(dy2), rows, n, out.data_ptr(), accumulate, partial.data_ptr(), s), "linear_bias_grad")
    return out
