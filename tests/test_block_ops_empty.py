"""Block operators on matrices without rows or columns. The sizes of scratch need no device: they are asked in a child process, which a
division by zero would end."""
import subprocess
import sys

import pytest
import torch

from parameter_server_b200._lib import C
from parameter_server_b200.ops import act8, linear, norm

gpu = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def test_scratch_of_nothing_is_nothing():
    calls = ["column_sum_scratch(4, 0)", "column_sum_scratch(0, 0)", "layer_norm_bwd_scratch(4, 0)", "layer_norm_bwd_scratch(0, 0)",
             "act8_wgrad_scratch(4, 0, 8)", "act8_wgrad_scratch(4, 8, 0)", "act8_wgrad_scratch(0, 8, 8)", "act8_wgrad_scratch(0, 0, 0)"]
    lines = ["from parameter_server_b200._lib import C"] + [f"print({c!r}, C.{c}, flush=True)" for c in calls]
    r = subprocess.run([sys.executable, "-c", "\n".join(lines)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.splitlines() == [f"{c} 0" for c in calls], (r.returncode, r.stdout, r.stderr[-300:])


def test_scratch_of_no_rows_still_holds_a_result():
    assert C.column_sum_scratch(0, 5) == 5 and C.layer_norm_bwd_scratch(0, 5) == 10


@gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_no_columns(dtype):
    x = torch.zeros(4, 0, dtype=dtype, device="cuda")
    for t in (x, x[:0], x.view(2, 2, 0)):
        got = linear.linear_bias_grad(t)
        assert got.shape == (0,) and got.dtype == F32
        out = torch.zeros(0, device="cuda")
        assert linear.linear_bias_grad(t, out=out, accumulate=True) is out
    stats = torch.zeros(4, device="cuda")
    dx, dw, db = norm.layer_norm_backward(x, x, None, stats, stats)
    assert dx.shape == (4, 0) and dw.shape == db.shape == (0,)
    kept = act8.act8_pack(x)
    assert kept.shape == (4, 0) and act8.act8_unpack(kept, dtype).shape == (4, 0)


@gpu
def test_products_with_an_empty_side():
    z = lambda *s: torch.zeros(*s, dtype=BF, device="cuda")  # noqa: E731
    for rows, n in ((4, 0), (0, 8), (0, 0)):
        y, h = linear.linear_act(z(rows, 16), z(n, 16), z(n), act="silu", residual=z(rows, n), save="act8")
        assert y.shape == (rows, n) and h.shape == (rows, n)
        assert linear.linear_act_dgrad(z(rows, 16), z(16, n), h, act="silu").shape == (rows, n)
        assert act8.act8_wgrad(z(rows, 16), h).shape == (16, n)
        assert act8.act8_wgrad(z(rows, n), act8.act8_pack(z(rows, 16))).shape == (n, 16)
