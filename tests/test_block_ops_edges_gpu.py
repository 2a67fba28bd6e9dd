"""Block operators where values, sizes or settings reach an edge: the largest steps of the 8-bit format on every way that the weight
gradient takes. Against 64 bits, with the bounds of ``test_block_ops_gpu``."""
import pytest
import torch

from parameter_server_b200._lib import C
from parameter_server_b200.ops import act8
from parameter_server_b200.ops import gemm as G

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def rand(*shape, seed=0, std=1.0, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * len(shape) + sum(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


# ---- the weight gradient from blocks with the format's largest steps --------------------------------------------------------

# converted tile by tile; unpacked first; on clusters
@pytest.mark.parametrize("way,T,N,K", [("converted", 4096, 1536, 2048), ("unpacked", 512, 4096, 4096), ("clusters", 300, 96, 160)])
def test_act8_wgrad_of_the_largest_steps(way, T, N, K):
    """Whole numbers times 2^112 (the last step at which 32896 steps are finite in 32 bits) to 2^122 (the largest a finite block has):
    every value is finite, and so is every sum. One more block is marked as not finite."""
    assert (C.act8_wgrad_scratch(T, N, K) == 0) == (way == "converted")
    gen = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randint(-63, 64, (T, K), generator=gen, device="cuda").to(torch.int8)   # 64 * 2^122 is no 32-bit number
    e = torch.zeros(T, -(-K // 512) * 16, dtype=torch.uint8, device="cuda")
    blocks = K // 32
    steps = torch.tensor([239, 240, 245, 249, 127], dtype=torch.uint8, device="cuda")
    e[:, :blocks] = steps[torch.arange(blocks, device="cuda") % 5]                      # one for all tokens of a column
    x8 = act8.Act8(q, e, K)
    dy = rand(T, N, std=2.0 ** -100)
    x = q.double() * torch.ldexp(torch.ones(K, dtype=torch.float64, device="cuda"), e[0, torch.arange(K, device="cuda") // 32].int() - 127)
    assert torch.equal(act8.act8_unpack(x8, F32).double(), x)
    got = act8.act8_wgrad(dy, x8)
    want = dy.double().t() @ x
    # chains of 512 tokens in the tensor core (34 cut sums of 2^-23), joined with one rounding each
    bound = (34 * 2.0 ** -23 + (T / 512 + 8) * 2.0 ** -24) * (dy.double().abs().t() @ x.abs()) + 2.0 ** -23 * want.abs()
    assert torch.isfinite(got).all() and ((got.double() - want).abs() <= bound).all()
    e[T // 2, 1], q[T // 2, 32:64] = 255, 0
    got2 = act8.act8_wgrad(dy, x8)
    assert torch.isnan(got2[:, 32:64]).all()
    got2[:, 32:64] = got[:, 32:64]
    assert torch.equal(got2, got)
    G.check_gemm_errors()
