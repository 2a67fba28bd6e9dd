"""Layer norm, forward and backward (``csrc/kernels/norm.cu``), with the normalised rows kept in 8 bits on request.

Rows are the last dimension of ``x`` (bf16 or fp32); weight and bias have its type and may be None. Statistics, sums and the
weight's gradients are fp32, and the latter are added in a fixed order: the same inputs give the same bits.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .._lib import C
from .act8 import Act8, _DTYPES, check, launch_stream, row_stride, rows2d


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _param(t: Optional[torch.Tensor], d: int, x: torch.Tensor, what: str, name: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.dtype != x.dtype or t.dim() != 1 or t.numel() != d or t.get_device() != x.get_device():
        raise ValueError(f"{what}: {name}: expected {d} values of {x.dtype} on {x.device}, got {tuple(t.shape)} of {t.dtype} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def _forward(x, weight, bias, eps, keep8, what):
    dt = _DTYPES.get(x.dtype)
    if dt is None:
        raise ValueError(f"{what}: bf16 or fp32, not {x.dtype}")
    s = launch_stream(x)
    x2 = rows2d(x, what)
    rows, d = x2.shape
    if d == 0:
        raise ValueError(f"{what}: rows of no columns have no mean")
    weight, bias = _param(weight, d, x, what, "weight"), _param(bias, d, x, what, "bias")
    y = torch.empty_like(x2) if x2.is_contiguous() else x2.new_empty((rows, d))
    rstd = x2.new_empty(rows, dtype=torch.float32)
    if keep8:
        kept, mean = Act8.for_rows(x2, d), None
        k = kept.args()
    else:
        kept, mean = None, torch.empty_like(rstd)
        k = (0, 0, 0, 0)
    check(C.layer_norm_fwd(dt, x2.data_ptr(), row_stride(x2), _ptr(weight), _ptr(bias), y.data_ptr(), d, _ptr(mean), rstd.data_ptr(), *k,
                           rows, d, eps, s), what)
    if x.dim() != 2:
        y = y.view(x.shape)
    return y, (kept if keep8 else mean), rstd


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(y, mean, rstd)``: ``y = (x - mean) * rstd * weight + bias`` over the last dimension; mean and rstd (fp32, one per row)
    are what ``layer_norm_backward`` needs beside ``x``."""
    return _forward(x, weight, bias, eps, False, "layer_norm")


def layer_norm_act8(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                    eps: float = 1e-5) -> Tuple[torch.Tensor, Act8, torch.Tensor]:
    """``(y, xhat8, rstd)``: as :func:`layer_norm`, with the normalised rows ``(x - mean) * rstd`` kept in 8 bits. The backward
    pass needs neither ``x`` nor the mean, and the linear layer that follows needs no copy of ``y`` for its weight gradient
    (``act8_wgrad`` with ``weight`` and ``bias``)."""
    return _forward(x, weight, bias, eps, True, "layer_norm_act8")


def _backward(dy, x, kept, weight, mean, rstd, residual_grad, weight_grad, bias_grad, accumulate, what):
    dt = _DTYPES.get(dy.dtype)
    if dt is None:
        raise ValueError(f"{what}: bf16 or fp32, not {dy.dtype}")
    s, dev = launch_stream(dy), dy.get_device()
    dy2 = rows2d(dy, what)
    rows, d = dy2.shape
    if x is not None:
        if x.shape != dy.shape or x.dtype != dy.dtype or x.get_device() != dev:
            raise ValueError(f"{what}: x and dy differ ({tuple(x.shape)} of {x.dtype}, {tuple(dy.shape)} of {dy.dtype})")
        x = rows2d(x, what)
    elif kept.rows != rows or kept.cols != d or kept.device_index != dev:
        raise ValueError(f"{what}: checkpoint of {kept.rows} x {kept.cols} on {kept.device}, dy of {rows} x {d} on {dy.device}")
    weight = _param(weight, d, dy, what, "weight")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t is not None and (t.dtype != torch.float32 or t.numel() != rows or t.get_device() != dev or not t.is_contiguous()):
            raise ValueError(f"{what}: {name} must be {rows} contiguous fp32 values on {dy.device}")
    join = None
    if residual_grad is not None:
        if residual_grad.shape != dy.shape or residual_grad.dtype != dy.dtype or residual_grad.get_device() != dev:
            raise ValueError(f"{what}: residual_grad must be like dy ({tuple(dy.shape)} of {dy.dtype})")
        join = rows2d(residual_grad, what)
    grads = []
    for name, t in (("weight_grad", weight_grad), ("bias_grad", bias_grad)):
        if t is None:
            if accumulate:
                raise ValueError(f"{what}: accumulate needs {name}")
            t = dy2.new_empty(d, dtype=torch.float32)
        elif t.dtype != torch.float32 or t.shape != (d,) or t.get_device() != dev or not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be {d} contiguous fp32 values on {dy.device}")
        grads.append(t)
    dx = torch.empty_like(dy2) if dy2.is_contiguous() else dy2.new_empty((rows, d))
    partial = dy2.new_empty(C.layer_norm_bwd_scratch(rows, d), dtype=torch.float32)
    check(C.layer_norm_bwd(dt, dy2.data_ptr(), row_stride(dy2), _ptr(x), 0 if x is None else row_stride(x),
                           *((0, 0, 0, 0) if kept is None else kept.args()), _ptr(weight), _ptr(mean), rstd.data_ptr(), _ptr(join),
                           0 if join is None else row_stride(join), dx.data_ptr(), d, grads[0].data_ptr(), grads[1].data_ptr(), accumulate,
                           partial.data_ptr(), rows, d, s), what)
    return (dx if dy.dim() == 2 else dx.view(dy.shape)), grads[0], grads[1]


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor, rstd: torch.Tensor, *,
                        residual_grad: Optional[torch.Tensor] = None, weight_grad: Optional[torch.Tensor] = None,
                        bias_grad: Optional[torch.Tensor] = None, accumulate: bool = False):
    """``(dx, weight_grad, bias_grad)`` of :func:`layer_norm`. ``residual_grad`` (like ``dy``) is added to dx: the gradient that
    reaches ``x`` past the norm. The weight's gradients are fp32; given buffers are written, or added to with ``accumulate``."""
    return _backward(dy, x, None, weight, mean, rstd, residual_grad, weight_grad, bias_grad, accumulate, "layer_norm_backward")


def layer_norm_act8_backward(dy: torch.Tensor, xhat8: Act8, weight: Optional[torch.Tensor], rstd: torch.Tensor, *,
                             residual_grad: Optional[torch.Tensor] = None, weight_grad: Optional[torch.Tensor] = None,
                             bias_grad: Optional[torch.Tensor] = None, accumulate: bool = False):
    """:func:`layer_norm_backward` from the 8-bit checkpoint of :func:`layer_norm_act8`."""
    return _backward(dy, None, xhat8, weight, None, rstd, residual_grad, weight_grad, bias_grad, accumulate, "layer_norm_act8_backward")
