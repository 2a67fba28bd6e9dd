"""The least limit for the waits inside the block operators' products, 0 s. The hardware keeps a thread that asks a barrier for a while,
so a wait that is answered in time still is; one that is not gives up. Either way the launch ends, what it reports is right (the result, or
the error word), and the next call is right."""
import pytest
import torch

from parameter_server_b200.ops import act8, linear
from parameter_server_b200.ops import gemm as G

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def rand(*shape, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * len(shape) + sum(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(BF)


def product(M, N, K):
    x, w = rand(M, K), rand(N, K, seed=1, std=K ** -0.5)
    return lambda **kw: linear.linear_act(x, w, act="silu", **kw)


def input_gradient(M, N, K):
    dy, w, h = rand(M, K), rand(K, N, seed=1, std=K ** -0.5), act8.act8_pack(rand(M, N, seed=2))
    return lambda **kw: linear.linear_act_dgrad(dy, w, h, act="silu", **kw)


def weight_gradient(T, N, K):
    dy, x8 = rand(T, N), act8.act8_pack(rand(T, K, seed=1))
    return lambda **kw: act8.act8_wgrad(dy, x8, **kw)


# pairs on whole tiles and on cut ones, clusters for few tokens; the weight gradient converted, unpacked, and on clusters
CALLS = [(product, 2048, 2048, 4096), (product, 300, 256, 65536), (product, 16, 2048, 16384), (input_gradient, 2048, 2048, 4096),
         (input_gradient, 64, 1024, 16384), (weight_gradient, 4096, 1536, 2048), (weight_gradient, 20000, 130, 40),
         (weight_gradient, 8192, 4096, 1024), (weight_gradient, 8192, 256, 256)]


@pytest.mark.parametrize("make,a,b,c", CALLS)
def test_a_wait_that_runs_out_is_reported_and_leaves_nothing_behind(make, a, b, c):
    call = make(a, b, c)
    want = call()
    G.check_gemm_errors()
    flush = torch.empty(64 << 20, device="cuda")
    for _ in range(4):
        flush.fill_(0.0)   # the operands come from memory
        got = call(wait_limit_s=0.0)
        try:
            G.check_gemm_errors()
        except RuntimeError as e:
            assert "bounded wait ran out (site " in str(e)
        else:
            assert torch.equal(got, want)
        assert torch.equal(call(), want)   # the next launch, and one beside another kernel
        other = rand(512, 512, seed=3)
        assert torch.equal(G.gemm(other, other), G.gemm(other, other)) and torch.equal(call(), want)
        G.check_gemm_errors()
