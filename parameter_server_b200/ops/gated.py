"""The gated feed-forward layer of a decoder block (``csrc/kernels/linear_fused.cuh``), bf16 operands and fp32 sums:

* ``gated_linear``: ``act(x wg^T + bg) * (x wu^T + bu)`` in one kernel, with both factors' values before the activation kept for the
  backward pass on request;
* ``gated_linear_dgrad``: the gradients that reach those values, ``da * u * act'(g)`` and ``da * act(g)`` side by side with ``da = dy w``,
  and ``act(g) * u`` again.

The layer behind is ``ops.linear.linear_act``. With both gradients in one matrix, the rest of the backward pass is the plain linear layer's:
``linear_act_dgrad(dh, w, None)``, ``ops.gemm.linear_wgrad(dh, x)`` or ``ops.act8.act8_wgrad(dh, x8)``, ``linear_bias_grad(dh)``.
A bounded wait that ran out is reported by ``ops.gemm.check_gemm_errors``.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .act8 import Act8, launch_stream, operand, row_stride, rows2d, vector
from .dropout import NO_DROPOUT
from .linear import _BIAS_TYPES, ACTIVATIONS, _act_code, _like, _run

Kept = Union[torch.Tensor, Tuple[Act8, Act8]]
_NONE_KEPT = (0,) * 8


def _rows(like: torch.Tensor, rows: int, cols: int):
    """An empty bf16 matrix with rows on 16-byte boundaries, and the elements between them (``act8.result`` in one step)."""
    ld = cols + 7 & -8
    return torch.empty_strided((rows, cols), (ld, 1), dtype=torch.bfloat16, device=like.device), ld


def _misfit(rows, cols, K, save):
    what = "gated_linear"
    if save not in (None, "bf16", "act8"):
        raise ValueError(f"{what}: save is None, 'bf16' or 'act8', not {save!r}")
    if rows % 2:
        raise ValueError(f"{what}: w has as many rows for the gate as for the other factor, not {rows} in all")
    if cols != K:
        raise ValueError(f"{what}: x has {K} columns, w has {cols}")
    raise ValueError(f"{what}: a sum over no columns")


def gated_linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, *, act: Optional[str] = "silu",
                 save: Optional[str] = None, out: Optional[torch.Tensor] = None, wait_limit_s: float = 2.0):
    """``act(g) * u`` with ``[g | u] = x w^T + bias`` for ``x`` ``[..., K]``, ``w`` ``[2F, K]`` (bf16; the gate's rows first) and ``bias``
    ``[2F]`` (bf16 or fp32); the result is ``[..., F]``. ``act``: "none", "relu", "gelu", "gelu_tanh" or "silu".

    ``save`` = "bf16" or "act8" also returns what :func:`gated_linear_dgrad` takes: ``(y, h)`` with ``h`` ``[..., 2F]`` in bf16, or two
    :class:`~.act8.Act8`, one of ``g`` and one of ``u``. ``out`` (bf16) receives ``y``; it must not overlap ``x`` or ``w``. Results whose
    rows are no multiple of 8 long have padded rows (``stride(-2)``), as the next product wants them."""
    what = "gated_linear"
    code = ACTIVATIONS.get(act)
    if code is None:
        _act_code(act, what)
    s, dev = launch_stream(x), x.get_device()
    x2, xp, ldx, _held = operand(x, "gated_linear x", dev)
    w, wp, ldw, _held_w = operand(w, "gated_linear w", dev)
    (M, K), (rows, cols) = x2.shape, w.shape
    F = rows >> 1
    if rows & 1 or cols != K or K == 0 or (save is not None and save != "bf16" and save != "act8"):
        _misfit(rows, cols, K, save)
    bp, b32 = 0, False
    if bias is not None:
        bp, b32 = vector(bias, 2 * F, _BIAS_TYPES, dev, "gated_linear: bias"), bias.dtype is torch.float32
    two = x.dim() == 2
    if out is None:
        y, ldy = _rows(x2, M, F)
    else:
        _like(out, x.shape[:-1] + (F,), dev, "gated_linear: out")
        y = out if out.dim() == 2 else out.view(M, F)
        if F > 1 and y.stride(1) != 1:
            raise ValueError(f"{what}: the values of a row of out must be contiguous")
        ldy = row_stride(y)
        if M > 1 and ldy < F:
            raise ValueError(f"{what}: rows of out lie on one another")
    h, hp, ldh, kept = None, 0, 0, _NONE_KEPT
    if save == "bf16":
        h, ldh = _rows(x2, M, 2 * F)
        hp = h.data_ptr()
    elif save == "act8":
        h = Act8.for_rows(x2, F), Act8.for_rows(x2, F)
        kept = h[0]._args + h[1]._args
    if M and F:
        _run(dev, s, what, (False, True, code, M, F, K, xp, ldx, wp, ldw, bp, b32, 0, 0, y.data_ptr(), ldy, 0, 0, hp, ldh, *kept, NO_DROPOUT), wait_limit_s)
    if out is not None:
        y = out
    elif not two:
        y = y.view(x.shape[:-1] + (F,))
    if save is None:
        return y
    return y, (h if two or save == "act8" else h.view(x.shape[:-1] + (2 * F,)))


def gated_linear_dgrad(dy: torch.Tensor, w: torch.Tensor, h: Kept, *, act: Optional[str] = "silu", recompute: bool = False,
                       wait_limit_s: float = 2.0):
    """``dh = [da * u * act'(g) | da * act(g)]``, ``[..., 2F]``, with ``da = dy w`` for ``dy`` ``[..., K]`` and the weight ``w`` ``[K, F]`` (as the
    forward pass has it: ``y = a w^T``) of the layer that took ``a = act(g) * u``; ``h`` is what ``gated_linear(save=...)`` returned. With
    ``recompute``: ``(dh, a)``, where ``a`` (bf16) is what the weight gradient of that layer needs."""
    what = "gated_linear_dgrad"
    code = ACTIVATIONS.get(act)
    if code is None:
        _act_code(act, what)
    s, dev = launch_stream(dy), dy.get_device()
    dy2, dyp, lddy, _held = operand(dy, "gated_linear_dgrad dy", dev)
    w, wp, ldw, _held_w = operand(w, "gated_linear_dgrad w", dev)
    (M, K), (rows, F) = dy2.shape, w.shape
    if rows != K:
        raise ValueError(f"{what}: dy has {K} columns, w has {rows} rows")
    if K == 0:
        raise ValueError(f"{what}: a sum over no columns")
    two = dy.dim() == 2
    pre, ldpre, kept = 0, 0, _NONE_KEPT
    if isinstance(h, torch.Tensor):
        _like(h, (M, 2 * F) if two else dy.shape[:-1] + (2 * F,), dev, "gated_linear_dgrad: h")
        h = rows2d(h, what)
        pre, ldpre = h.data_ptr(), row_stride(h)
    elif isinstance(h, (tuple, list)) and len(h) == 2 and isinstance(h[0], Act8) and isinstance(h[1], Act8):
        for k in h:
            if k.rows != M or k.cols != F or k.device_index != dev:
                raise ValueError(f"{what}: checkpoint of {k.rows} x {k.cols} on {k.device}, expected {M} x {F} on {dy.device}")
        kept = h[0]._args + h[1]._args
    else:
        raise ValueError(f"{what}: h is what gated_linear(save=...) returned, not {type(h).__name__}")
    dh, ld = _rows(dy2, M, 2 * F)
    a, lda = _rows(dy2, M, F) if recompute else (None, 0)
    if M and F:
        _run(dev, s, what, (True, True, code, M, F, K, dyp, lddy, wp, ldw, 0, False, 0, 0, dh.data_ptr(), ld, 0 if a is None else a.data_ptr(), lda,
                            pre, ldpre, *kept, NO_DROPOUT), wait_limit_s)
    if not two:
        dh = dh.view(dy.shape[:-1] + (2 * F,))
        a = None if a is None else a.view(dy.shape[:-1] + (F,))
    return (dh, a) if recompute else dh
