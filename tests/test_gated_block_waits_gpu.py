"""The least limit for the waits inside the gated layer's products and the linear layer's with dropout, 0 s (`test_block_ops_waits_gpu.py`
says what that does): a wait that runs out is reported, and leaves the next calls right."""
import pytest
import torch
from test_block_ops_waits_gpu import rand

from parameter_server_b200.ops import act8, gated, linear
from parameter_server_b200.ops import gemm as G

pytestmark = pytest.mark.gpu


def forward(M, N, K, save=None):
    x, w = rand(M, K), rand(2 * N, K, seed=1, std=K ** -0.5)
    first = (lambda y: y) if save is None else (lambda y: y[0])
    return lambda **kw: first(gated.gated_linear(x, w, save=save, **kw))


def backward(M, N, K, bits):
    dy, w, h = rand(M, K), rand(K, N, seed=1, std=K ** -0.5), rand(M, 2 * N, seed=2)
    if bits == 8:
        h = act8.act8_pack(h[:, :N]), act8.act8_pack(h[:, N:])
    return lambda **kw: gated.gated_linear_dgrad(dy, w, h, **kw)


def dropped(M, N, K, seed):
    x, w, r = rand(M, K), rand(N, K, seed=1, std=K ** -0.5), rand(M, N, seed=2)
    seed = torch.tensor([seed], device="cuda") if seed else 7
    return lambda **kw: linear.linear_act(x, w, residual=r, dropout=(0.1, seed, 3), **kw)


# pairs on whole tiles (several to a pair) and on cut ones, clusters for few tokens
CALLS = [(forward, 4096, 2048, 4096), (forward, 4096, 2048, 1024, "bf16"), (forward, 5000, 250, 12300, "act8"), (forward, 16, 2048, 16384, "act8"),
         (backward, 4096, 2048, 4096, 16), (backward, 8192, 2048, 1024, 8), (backward, 40000, 128, 1024, 8), (backward, 10000, 250, 12300, 16), (backward, 64, 1024, 16384, 8),
         (dropped, 4096, 2048, 4096, 0), (dropped, 2048, 2048, 4096, 5), (dropped, 5000, 500, 12300, 0), (dropped, 16, 2048, 16384, 5)]


@pytest.mark.parametrize("make,sizes", [(c[0], c[1:]) for c in CALLS])
def test_a_wait_that_runs_out_is_reported_and_leaves_nothing_behind(make, sizes):
    call = make(*sizes)
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
