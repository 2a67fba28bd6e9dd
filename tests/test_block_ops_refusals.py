"""Calls that the block operators refuse before anything is launched. On a machine without a GPU: what is checked ahead of the device."""
import pytest
import torch

from parameter_server_b200.ops import act8, linear, norm

BF = torch.bfloat16
gpu = pytest.mark.gpu


def test_host_tensors_are_refused():
    x = torch.zeros(4, 32, dtype=BF)
    for call in (lambda: norm.layer_norm(x), lambda: norm.layer_norm_act8(x), lambda: act8.act8_pack(x), lambda: linear.linear_act(x, x),
                 lambda: linear.linear_act_dgrad(x, x, x, act="relu"), lambda: linear.linear_bias_grad(x),
                 lambda: norm.layer_norm_backward(x, x, None, torch.zeros(4), torch.zeros(4))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_checkpoint_layout_is_checked():
    q, e = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 16, dtype=torch.uint8)
    a = act8.Act8(q, e, 50)
    assert a.shape == (4, 50) and a.nbytes == 4 * 80
    assert act8.Act8(torch.zeros(8, 80, dtype=torch.int8)[:, 16:80], torch.zeros(8, 16, dtype=torch.uint8), 64).rows == 8
    for bad in ((q.float(), e, 50), (q, e.to(torch.int8), 50), (q[0], e, 50), (q, e[:3], 50), (q, e, 65), (q, e[:, :1], 50), (q, e, -1),
                (torch.zeros(4, 40, dtype=torch.int8), e, 40), (q[:, 1:], e, 40), (torch.zeros(64, 4, dtype=torch.int8).t(), e, 4)):
        with pytest.raises(ValueError, match="Act8"):
            act8.Act8(*bad)
    assert act8.Act8.empty(3, 40, "cpu").q.shape == (3, 48) and act8.Act8.empty(3, 40, "cpu").e.shape == (3, 16)


@gpu
def test_types_shapes_and_names_are_refused():
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    x, w, f = z(8, 64), z(32, 64), z(64, dtype=torch.float32)
    x8 = act8.act8_pack(x)
    stats = z(8, dtype=torch.float32)
    refused = [
        lambda: norm.layer_norm(x.half()), lambda: norm.layer_norm(x, f), lambda: norm.layer_norm(x, z(63)), lambda: norm.layer_norm(x, z(64), z(1, 64)),
        lambda: norm.layer_norm(z(8, 0)), lambda: norm.layer_norm(z(())),
        lambda: norm.layer_norm_backward(x, z(8, 63), None, stats, stats), lambda: norm.layer_norm_backward(x, x.float(), None, stats, stats),
        lambda: norm.layer_norm_backward(x, x, None, stats[:7], stats), lambda: norm.layer_norm_backward(x, x, None, stats, stats.double()),
        lambda: norm.layer_norm_backward(x, x, None, stats, stats, residual_grad=x.float()), lambda: norm.layer_norm_backward(x, x, None, stats, stats, accumulate=True),
        lambda: norm.layer_norm_backward(x, x, None, stats, stats, weight_grad=z(64)), lambda: norm.layer_norm_act8_backward(z(9, 64), x8, None, stats),
        lambda: act8.act8_pack(x.half()), lambda: act8.act8_unpack(x8, torch.float16),
        lambda: linear.linear_act(x, z(32, 63)), lambda: linear.linear_act(x.float(), w), lambda: linear.linear_act(x, w, act="tanh"),
        lambda: linear.linear_act(x, w, save="int8"), lambda: linear.linear_act(x, w, z(31)), lambda: linear.linear_act(x, w, residual=z(8, 31)),
        lambda: linear.linear_act(x, w, residual=z(8, 32, dtype=torch.float32)), lambda: linear.linear_act(x, w, out=z(8, 33)),
        lambda: linear.linear_act(x, w, out=z(32, 8).t()), lambda: linear.linear_act(z(8, 0), z(32, 0)), lambda: linear.linear_act(x, w.cpu()),
        lambda: linear.linear_act_dgrad(x, z(63, 32), z(8, 32), act="relu"), lambda: linear.linear_act_dgrad(x, z(64, 32), None, act="relu"),
        lambda: linear.linear_act_dgrad(x, z(64, 32), z(8, 31), act="relu"), lambda: linear.linear_act_dgrad(x, z(64, 32), x8, act="relu"),
        lambda: linear.linear_bias_grad(x.half()), lambda: linear.linear_bias_grad(x, out=z(64)), lambda: linear.linear_bias_grad(x, accumulate=True),
        lambda: act8.act8_wgrad(z(9, 32), x8), lambda: act8.act8_wgrad(z(8, 32).float(), x8), lambda: act8.act8_wgrad(z(8, 32), x8, bias=z(64)),
        lambda: act8.act8_wgrad(z(8, 32), x8, weight=z(63)), lambda: act8.act8_wgrad(z(8, 32), x8, bias=z(64), dy_sum=f),
        lambda: act8.act8_wgrad(z(8, 32), x8, out=z(32, 64)), lambda: act8.act8_wgrad(z(8, 32), x8, accumulate=True),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    torch.cuda.synchronize()
