"""Linear layers of a decoder block with their neighbours in the epilogue."""
from __future__ import annotations

from typing import Optional

import torch

from .._lib import C
from .act8 import _DTYPES, check, launch_stream, row_stride, rows2d


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
        out = torch.empty(n, dtype=torch.float32, device=dy.device)
    elif out.dtype != torch.float32 or out.shape != (n,) or out.device != dy.device or not out.is_contiguous():
        raise ValueError(f"linear_bias_grad: out must be {n} contiguous fp32 values on {dy.device}")
    partial = torch.empty(C.column_sum_scratch(rows, n), dtype=torch.float32, device=dy.device)
    check(C.column_sum(dt, dy2.data_ptr(), row_stride(dy2), rows, n, out.data_ptr(), accumulate, partial.data_ptr(), s), "linear_bias_grad")
    return out
