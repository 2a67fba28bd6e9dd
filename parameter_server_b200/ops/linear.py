"""Linear layers of a decoder block with their neighbours in the epilogue (``csrc/kernels/linear_fused.cuh``), bf16 operands and
fp32 sums:

* ``linear_act``: ``act(x w^T + b) + residual``, with the value before the activation kept for the backward pass;
* ``linear_act_dgrad``: the gradient that reaches that value, ``(dy w) * act'(h)``, and ``act(h)`` again;
* ``linear_bias_grad``: the sum of dy's rows in a fixed order.

The weight gradient is ``ops.gemm.linear_wgrad``, or ``ops.act8.act8_wgrad`` from an 8-bit checkpoint. A bounded wait that ran out
is reported by ``ops.gemm.check_gemm_errors``.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from .._lib import C
from .act8 import _DTYPES, _ld, _matrix, Act8, check, launch_stream, row_stride, rows2d
from .gemm import _err_flag, workspace

ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


def _act_code(act, what: str) -> int:
    code = ACTIVATIONS.get(act)
    if code is None:
        raise ValueError(f"{what}: act is one of {sorted(k for k in ACTIVATIONS if k)}, not {act!r}")
    return code


def _launch(dgrad, act, M, N, K, a, w, bias, residual, out, out2, pre, kept, limit, s, what, scratch=0):
    rc = C.linear_fused(dgrad, act, M, N, K, a.data_ptr(), _ld(a), w.data_ptr(), _ld(w),
                        0 if bias is None else bias.data_ptr(), bias is not None and bias.dtype == torch.float32,
                        0 if residual is None else residual.data_ptr(), 0 if residual is None else row_stride(residual),
                        out.data_ptr(), row_stride(out), 0 if out2 is None else out2.data_ptr(), N,
                        0 if pre is None else pre.data_ptr(), 0 if pre is None else row_stride(pre),
                        *((0, 0, 0, 0) if kept is None else kept.args()),
                        scratch, _err_flag(a.device).data_ptr(), limit, s)
    if rc == C.NEEDS_WORKSPACE and scratch == 0:   # only where tiles are cut along the contraction
        scratch = workspace(a.get_device(), s)
        return _launch(dgrad, act, M, N, K, a, w, bias, residual, out, out2, pre, kept, limit, s, what, scratch.data_ptr())
    check(rc, what)


def linear_act(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None, *, act: Optional[str] = None,
               residual: Optional[torch.Tensor] = None, save: Optional[str] = None, out: Optional[torch.Tensor] = None,
               wait_limit_s: float = 2.0):
    """``act(x w^T + bias) + residual`` for ``x`` ``[..., K]``, ``w`` ``[N, K]`` (bf16), ``bias`` ``[N]`` (bf16 or fp32) and
    ``residual`` ``[..., N]`` (bf16). ``act``: "none", "relu", "gelu", "gelu_tanh" or "silu".

    ``save`` = "bf16" or "act8" also returns ``h = x w^T + bias`` as :func:`linear_act_dgrad` takes it: ``(y, h)`` with ``h`` a bf16
    tensor like ``y``, or an :class:`~.act8.Act8`. ``out`` (bf16, may be ``residual`` itself) receives ``y``."""
    what = "linear_act"
    code = _act_code(act, what)
    if save not in (None, "bf16", "act8"):
        raise ValueError(f"{what}: save is None, 'bf16' or 'act8', not {save!r}")
    s = launch_stream(x)
    x2, w = _matrix(x, f"{what} x"), _matrix(w, f"{what} w", x)
    M, K = x2.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"{what}: x has {K} columns, w has {w.shape[1]}")
    if K == 0:
        raise ValueError(f"{what}: a sum over no columns")
    if bias is not None and (bias.shape != (N,) or bias.dtype not in (torch.bfloat16, torch.float32) or bias.device != x.device
                             or not bias.is_contiguous()):
        raise ValueError(f"{what}: bias must be {N} contiguous bf16 or fp32 values on {x.device}")
    lead = x.shape[:-1]
    if residual is not None:
        if residual.shape != lead + (N,) or residual.dtype != torch.bfloat16 or residual.device != x.device:
            raise ValueError(f"{what}: residual must be {tuple(lead) + (N,)} bf16 on {x.device}")
        r2 = rows2d(residual, what)
    else:
        r2 = None
    if out is None:
        y = x2.new_empty((M, N))
    else:
        if out.shape != lead + (N,) or out.dtype != torch.bfloat16 or out.device != x.device:
            raise ValueError(f"{what}: out must be {tuple(lead) + (N,)} bf16 on {x.device}")
        y = out if out.dim() == 2 else out.view(M, N)
        if N > 1 and y.stride(1) != 1:
            raise ValueError(f"{what}: the values of a row of out must be contiguous")
    pre = x2.new_empty((M, N)) if save == "bf16" else None
    kept = Act8.for_rows(y, N) if save == "act8" else None
    if M and N:
        _launch(False, code, M, N, K, x2, w, bias, r2, y, None, pre, kept, wait_limit_s, s, what)
    if out is not None:
        y = out
    elif x.dim() != 2:
        y = y.view(*lead, N)
    if save is None:
        return y
    return y, (kept if pre is None else pre.view(*lead, N))


def linear_act_dgrad(dy: torch.Tensor, w: torch.Tensor, h: Union[torch.Tensor, Act8, None], *, act: Optional[str] = None,
                     recompute: bool = False, wait_limit_s: float = 2.0):
    """``(dy w) * act'(h)`` for ``dy`` ``[..., K]`` and the weight ``w`` ``[K, N]`` (as the forward pass has it: ``y = a w^T``) of the
    layer that took ``a = act(h)``; ``h`` ``[..., N]`` is what ``linear_act(save=...)`` returned (None where ``act`` is "none").
    With ``recompute``: ``(dh, a)``, where ``a`` (bf16) is what the weight gradient of that layer needs."""
    what = "linear_act_dgrad"
    code = _act_code(act, what)
    s = launch_stream(dy)
    dy2, w = _matrix(dy, f"{what} dy"), _matrix(w, f"{what} w", dy)
    M, K = dy2.shape
    N = w.shape[1]
    if w.shape[0] != K:
        raise ValueError(f"{what}: dy has {K} columns, w has {w.shape[0]} rows")
    if K == 0:
        raise ValueError(f"{what}: a sum over no columns")
    lead = dy.shape[:-1]
    pre = kept = None
    if isinstance(h, Act8):
        if h.rows != M or h.cols != N or h.device != dy.device:
            raise ValueError(f"{what}: checkpoint of {h.rows} x {h.cols} on {h.device}, expected {M} x {N} on {dy.device}")
        kept = h
    elif h is not None:
        if h.shape != lead + (N,) or h.dtype != torch.bfloat16 or h.device != dy.device:
            raise ValueError(f"{what}: h must be {tuple(lead) + (N,)} bf16 on {dy.device}")
        pre = rows2d(h, what)
    elif code != 0 or recompute:
        raise ValueError(f"{what}: h is needed")
    dh = dy2.new_empty((M, N))
    a = dy2.new_empty((M, N)) if recompute else None
    if M and N:
        _launch(True, code, M, N, K, dy2, w, None, None, dh, a, pre, kept, wait_limit_s, s, what)
    if dy.dim() != 2:
        dh = dh.view(*lead, N)
        a = None if a is None else a.view(*lead, N)
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
