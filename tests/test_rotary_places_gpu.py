"""Where rotary positions read and write: queries and keys whose heads share memory, and results that do."""
import pytest
import torch

from parameter_server_b200.ops import rotary

BF, F32 = torch.bfloat16, torch.float32
# [batch, tokens, heads, dim] with these strides, each a window on the same memory as its neighbours'
SHARED = [((1, 4, 3, 8), (0, 1, 8, 1)), ((2, 16, 3, 8), (128, 1, 16, 1)), ((1, 3, 2, 16), (0, 1, 9, 1)), ((2, 9, 4, 8), (2, 1, 100, 1)), ((1, 5, 4, 8), (0, 8, 8, 1)), ((2, 3, 4, 8), (0, 4, 0, 1)),
          ((3, 4, 1, 6), (1, 1, 1, 1)), ((2, 4, 2, 1), (8, 2, 1, 5))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("shape,strides", SHARED)
def test_heads_that_share_memory(shape, strides, dtype):
    base = torch.randn(4096, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    q = base.as_strided(shape, strides)
    k = base.as_strided(shape, strides, 7)
    freqs = torch.linspace(0.3, 1.0, shape[-1] // 2, dtype=torch.float64, device="cuda")
    for call in (rotary.rotary, rotary.rotary_backward):
        for got, want in zip(call(q, k, freqs), call(q.contiguous(), k.contiguous(), freqs)):
            assert torch.equal(got, want)
        three = call(q[0], None, freqs)
        assert torch.equal(three, call(q[0].contiguous(), None, freqs))
