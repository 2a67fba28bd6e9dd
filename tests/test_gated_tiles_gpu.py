"""The products of a gated layer, and the linear layer with dropout, on many whole tiles of CTA pairs, value by value against 64 bits
(`test_gated_gpu.py` has the bounds, and the sizes that go to the kernel for few tokens, to tiles with edges and to tiles that are cut).

Which kernel: up to 128 rows the one for few, above by the number of tiles: pairs take 256 rows by 256 columns (128 where there are at most 128;
a gated forward tile has 128 of each factor) and share 74 places, so that with more tiles some pairs have several, one after the other, whose
neighbours are asked for a tile ahead. Sums of fewer than 64 k-steps are never cut."""
import philox64
import pytest
import torch
from test_gated_gpu import ACTS, BF, F32, gated64, kept_is, near, phi, rand, sum_slack

from parameter_server_b200.ops import act8, gated, linear
from parameter_server_b200.ops import gemm as G

pytestmark = pytest.mark.gpu


# rows x columns x sum: tiles of 256 with a last column of tiles that is no whole one, with more than one tile to a pair (17 x 5 = 85, 33 x 4 = 132);
# of 128 with a whole and a half column (157 x 1, two units of a warp); whole ones only
DGRAD = [(4200, 1120, 136), (8200, 1000, 264), (40000, 128, 64), (40000, 96, 72), (5120, 1024, 192)]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", DGRAD)
def test_gated_backward_on_whole_tiles(M, N, K, act):
    dy, w = rand(M, K), rand(K, N, seed=1, std=K ** -0.5)
    da = dy.double() @ w.double()
    s = sum_slack(dy.double(), w.double())
    # every block of 32 and every row has a step of its own, so that none can stand for another
    h = (rand(M, 2 * N, seed=2).float() * torch.exp2(torch.randint(-6, 3, (M, 2 * N // 32), generator=torch.Generator(device="cuda").manual_seed(M), device="cuda").float()).repeat_interleave(32, 1)
         if N % 32 == 0 else rand(M, 2 * N, seed=2).float() * torch.exp2((torch.arange(M, device="cuda") % 9 - 6).float())[:, None]).to(BF)
    packed = act8.act8_pack(h[:, :N]), act8.act8_pack(h[:, N:])
    for kept, value in ((h, h.double()), (packed, torch.cat([act8.act8_unpack(k, F32).double() for k in packed], 1))):
        g, u = value[:, :N], value[:, N:]
        p = phi(g, act)
        dh, a = gated.gated_linear_dgrad(dy, w, kept, act=act, recompute=True)
        near(dh[:, :N], da * u * phi(g, act, slope=True), 1.2 * s * u.abs() + 2.0 ** -18 * (da * u).abs() * (1 + g.abs()))
        near(dh[:, N:], da * p, s * p.abs() + 2.0 ** -18 * da.abs() * (1 + g.abs()))
        near(a, p * u, 2.0 ** -18 * u.abs() * (1 + g.abs()))
        assert torch.equal(gated.gated_linear_dgrad(dy, w, kept, act=act), dh)
    G.check_gemm_errors()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", [(4200, 1120, 136), (8200, 1000, 264), (5120, 1024, 192)])
def test_gated_forward_on_whole_tiles(M, N, K, act):
    x, w, b = rand(M, K), rand(2 * N, K, seed=1, std=K ** -0.5), rand(2 * N, seed=2)
    want, slack, h, sh = gated64(x, w, b, act)
    y, pre = gated.gated_linear(x, w, b, act=act, save="bf16")
    near(pre, h, sh)
    near(y, want, slack)
    y8, (g8, u8) = gated.gated_linear(x, w, b.float(), act=act, save="act8")
    assert torch.equal(y8, y) and torch.equal(gated.gated_linear(x, w, b, act=act), y)
    kept_is(g8, h[:, :N], sh[:, :N])
    kept_is(u8, h[:, N:], sh[:, N:])
    G.check_gemm_errors()


@pytest.mark.parametrize("act", ["none", "relu", "gelu_tanh"])
@pytest.mark.parametrize("M,N,K", [(4200, 1120, 136), (8200, 1000, 264), (40000, 128, 64)])
def test_linear_with_dropout_on_whole_tiles(M, N, K, act):
    x, w, b, r = rand(M, K), rand(N, K, seed=1, std=K ** -0.5), rand(N, seed=2), rand(M, N, seed=3)
    seed, offset, p = 0xFEDCBA9876543210, (1 << 35) + 9, 0.35
    at = torch.tensor([seed - (1 << 64)], device="cuda")
    mask = torch.from_numpy(philox64.kept(M, N, p, seed, offset)).cuda()
    h = x.double() @ w.double().t() + b.double()
    v = phi(h, act)
    slack = philox64.grown(p) * (1.2 * (sum_slack(x.double(), w.double().t()) + 2.0 ** -23 * h.abs()) + 2.0 ** -19 * (1 + h.abs()))
    want, slack = torch.where(mask, philox64.grown(p) * v, 0.0), torch.where(mask, slack, 0.0)
    y, h8 = linear.linear_act(x, w, b, act=act, residual=r, save="act8", dropout=(p, seed, offset))
    near(y, want + r.double(), slack + 2.0 ** -22 * (want.abs() + r.double().abs()))
    kept_is(h8, h, sum_slack(x.double(), w.double().t()) + 2.0 ** -23 * h.abs())
    assert torch.equal(linear.linear_act(x, w, b, act=act, residual=r, dropout=(p, at, offset)), y)
    alone = linear.linear_act(x, w, b, act=act, dropout=(p, seed, offset))
    near(alone, want, slack + 2.0 ** -22 * want.abs())
    assert torch.equal(linear.linear_act(x, w, b, act=act, dropout=(p, at, offset)), alone) and (alone[~mask] == 0).all()
    G.check_gemm_errors()
