"""Calls that the gated block's operators refuse before anything is launched, and what they compute on the host."""
import math
import re
from pathlib import Path

import numpy as np
import philox64
import pytest
import torch

from parameter_server_b200.ops import act8, dropout, gated, linear, rotary

BF = torch.bfloat16
gpu = pytest.mark.gpu


def test_the_generator_has_its_published_answers():
    one = 0xFFFFFFFF
    for counter, key, want in [
        ((0, 0, 0, 0), (0, 0), "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
        ((one,) * 4, (one,) * 2, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
        ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), "d16cfe09 94fdcceb 5001e420 24126ea1"),
    ]:
        got = philox64.rounds(tuple(np.array([c]) for c in counter), key)
        assert " ".join(f"{int(w[0]):08x}" for w in got) == want


def test_host_tensors_are_refused():
    x, f = torch.zeros(2, 3, 8, dtype=BF), torch.ones(4, dtype=torch.float64)
    for call in (lambda: dropout.dropout(x, 0.1, 1), lambda: dropout.dropout_backward(x, 0.1, 1), lambda: rotary.rotary(x, x, f), lambda: rotary.rotary_backward(x, None, f),
                 lambda: gated.gated_linear(x, x), lambda: gated.gated_linear_dgrad(x, x, x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_launches_that_overlap_their_predecessor_read_coherently():
    """A non-coherent load is defined only for memory that nothing writes while the kernel runs; these may begin before their predecessor
    has ended, or put their result in their input's place."""
    for name in ("dropout.cu", "rotary.cu", "philox.cuh", "unaligned.cuh", "linear_fused.cuh", "linear_few.cuh"):
        text = (Path(dropout.__file__).parent.parent / "csrc" / "kernels" / name).read_text()
        assert not re.search(r"ld_nc|ld\.global\.nc|__ldg\(|__restrict__", text), name


def test_seeds_are_whole_numbers():
    assert dropout.drop_args(0.5, np.int64(-5), np.int32(3), 0, "dropout")[:3] == ((1 << 64) - 5, 0, 3)
    for seed, offset in ((0.5, 0), (1, 0.5), ("1", 0)):
        with pytest.raises(TypeError):
            dropout.drop_args(0.5, seed, offset, 0, "dropout")


@pytest.mark.parametrize("p", [-0.1, 1.0, 1.5, math.nan, 1 - 2.0 ** -40])
def test_shares_that_leave_nothing_are_refused(p):
    with pytest.raises(ValueError):
        dropout.drop_args(p, 1, 0, 0, "dropout")


def test_seeds_and_offsets_of_64_bits():
    for seed, offset in ((1 << 64, 0), (-(1 << 63) - 1, 0), (0, -1), (0, 1 << 64)):
        with pytest.raises(ValueError):
            dropout.drop_args(0.5, seed, offset, 0, "dropout")
    assert dropout.drop_args(0.5, -1, (1 << 64) - 1, 0, "dropout") == ((1 << 64) - 1, 0, (1 << 64) - 1, 1 << 31, 2.0)
    assert dropout.drop_args(0.0, 7, 0, 0, "dropout")[3:] == (0, 1.0)
    for seed in (torch.zeros(1), torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="seed"):
            dropout.drop_args(0.5, seed, 0, 0, "dropout")


def test_frequencies():
    f, scale = rotary.rotary_frequencies(8, 100.0, device="cpu")
    assert scale == 1.0 and f.dtype is torch.float64 and torch.allclose(f, 100.0 ** (-torch.arange(4, dtype=torch.float64) / 4), rtol=1e-14)
    linear, _ = rotary.rotary_frequencies(8, 100.0, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(linear, f / 4)
    ntk, _ = rotary.rotary_frequencies(8, 100.0, scaling="ntk", factor=4.0, device="cpu")
    assert ntk[0] == 1 and abs(ntk[3].item() * 4 / f[3].item() - 1) < 1e-12
    assert torch.allclose(rotary.rotary_frequencies(2, scaling="ntk", factor=4.0, device="cpu")[0], torch.tensor([0.25], dtype=torch.float64))
    yarn, grown = rotary.rotary_frequencies(64, scaling="yarn", factor=8.0, trained_length=4096, device="cpu")
    plain, _ = rotary.rotary_frequencies(64, device="cpu")
    turns = plain * 4096 / (2 * math.pi)
    assert abs(grown - (0.1 * math.log(8.0) + 1)) < 1e-15
    assert torch.equal(yarn[turns >= 32], plain[turns >= 32]) and torch.equal(yarn[turns <= 1], plain[turns <= 1] / 8)
    assert ((yarn <= plain) & (yarn >= plain / 8)).all() and (turns < 1).any() and (turns > 32).any()
    for bad in (dict(dim=0), dict(dim=7), dict(dim=8, base=0.0), dict(dim=8, factor=0.5), dict(dim=8, scaling="yarn", factor=2.0), dict(dim=8, scaling="log"),
                dict(dim=8, scaling="yarn", factor=2.0, trained_length=64, fast=1.0, slow=1.0)):
        with pytest.raises(ValueError, match="rotary_frequencies"):
            rotary.rotary_frequencies(**bad, device="cpu")


@gpu
def test_types_and_shapes_of_dropout_are_refused():
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    x = z(8, 64)
    refused = [
        lambda: dropout.dropout(x.half(), 0.1, 1), lambda: dropout.dropout(x, 0.1, 1, residual=z(8, 63)), lambda: dropout.dropout(x, 0.1, 1, residual=x.float()),
        lambda: dropout.dropout(x, 0.1, 1, residual=x.cpu()), lambda: dropout.dropout(x, 0.1, 1, out=z(9, 64)), lambda: dropout.dropout(x, 0.1, 1, out=x.float()),
        lambda: dropout.dropout(x, 0.1, 1, out=z(64, 8).t()), lambda: dropout.dropout(x, 1.0, 1), lambda: dropout.dropout(x, 0.1, z(1, dtype=torch.int32)),
        lambda: dropout.dropout(x, 0.1, torch.zeros(1, dtype=torch.int64)), lambda: dropout.dropout(x, 0.1, 1, out=z(1, 64).expand(8, 64)), lambda: dropout.dropout(z(()), 0.1, 1), lambda: dropout.dropout_backward(x, -0.5, 1),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    torch.cuda.synchronize()


@gpu
def test_types_and_shapes_of_rotary_are_refused():
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    q, k, f = z(2, 3, 4, 16), z(2, 3, 1, 16), z(8, dtype=torch.float64)
    pos = torch.arange(3, device="cuda")
    refused = [
        lambda: rotary.rotary(q.half(), None, f), lambda: rotary.rotary(z(3, 16), None, f), lambda: rotary.rotary(z(1, 2, 3, 4, 16), None, f),
        lambda: rotary.rotary(q, k[0], f), lambda: rotary.rotary(q, z(2, 4, 1, 16), f), lambda: rotary.rotary(q, z(2, 3, 1, 18), f), lambda: rotary.rotary(q, k.float(), f),
        lambda: rotary.rotary(q, k.cpu(), f), lambda: rotary.rotary(q, k, f.float()), lambda: rotary.rotary(q, k, f.cpu()), lambda: rotary.rotary(q, k, z(9, dtype=torch.float64)),
        lambda: rotary.rotary(q, k, z(16, dtype=torch.float64)[::2]), lambda: rotary.rotary(q, k, f, pos.float()), lambda: rotary.rotary(q, k, f, pos[:2]),
        lambda: rotary.rotary(q, k, f, pos.cpu()), lambda: rotary.rotary(q, k, f, pos.expand(3, 3)), lambda: rotary.rotary(q, k, f, out_q=z(2, 3, 4, 17)),
        lambda: rotary.rotary(q, None, f, out_k=k), lambda: rotary.rotary(q, k, f, out_q=z(2, 3, 1, 16).expand(2, 3, 4, 16)), lambda: rotary.rotary(q, k, f, pos.view(1, 1, 3)), lambda: rotary.rotary(q, k, f, out_k=z(2, 3, 16, 2).transpose(2, 3)[:, :, :1]), lambda: rotary.rotary_backward(q, k, f, out_q=q.float()),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    torch.cuda.synchronize()


@gpu
def test_types_and_shapes_of_the_gated_layer_are_refused():
    z = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    x, w, w2, h = z(8, 64), z(32, 64), z(64, 16), z(8, 32)
    x8, wide8 = act8.act8_pack(z(8, 16)), act8.act8_pack(z(8, 32))
    refused = [
        lambda: gated.gated_linear(x, z(32, 63)), lambda: gated.gated_linear(x, z(31, 64)), lambda: gated.gated_linear(x.float(), w), lambda: gated.gated_linear(x, w.float()),
        lambda: gated.gated_linear(x, w, act="tanh"), lambda: gated.gated_linear(x, w, save="int8"), lambda: gated.gated_linear(x, w, z(16)), lambda: gated.gated_linear(x, w, z(32).half()),
        lambda: gated.gated_linear(x, w, out=z(8, 32)), lambda: gated.gated_linear(x, w, out=z(8, 16, dtype=torch.float32)), lambda: gated.gated_linear(x, w, out=z(16, 8).t()), lambda: gated.gated_linear(x, w, out=z(1, 16).expand(8, 16)),
        lambda: gated.gated_linear(z(8, 0), z(32, 0)), lambda: gated.gated_linear(x, w.cpu()),
        lambda: gated.gated_linear_dgrad(x, z(63, 16), h), lambda: gated.gated_linear_dgrad(x, w2, z(8, 16)), lambda: gated.gated_linear_dgrad(x, w2, h.float()),
        lambda: gated.gated_linear_dgrad(x, w2, None), lambda: gated.gated_linear_dgrad(x, w2, x8), lambda: gated.gated_linear_dgrad(x, w2, (x8, wide8)),
        lambda: gated.gated_linear_dgrad(x, w2, (x8,)), lambda: gated.gated_linear_dgrad(x, w2, (h, h)), lambda: gated.gated_linear_dgrad(x, w2, h, act="swish"),
        lambda: gated.gated_linear_dgrad(z(9, 64), w2, (x8, x8)), lambda: gated.gated_linear_dgrad(z(8, 0), z(0, 16), h),
        lambda: linear.linear_act(x, w, dropout=(1.0, 1, 0)), lambda: linear.linear_act(x, w, dropout=(0.5, 1 << 64, 0)), lambda: linear.linear_act(x, w, dropout=(0.5, 1, -1)),
        lambda: linear.linear_act(x, w, dropout=(0.5, torch.zeros(1, dtype=torch.int64), 0)), lambda: linear.linear_act(x, w, dropout=0.5), lambda: linear.linear_act(x, w, dropout=(0.5, 1)),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    torch.cuda.synchronize()
