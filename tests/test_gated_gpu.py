"""The gated feed-forward layer, and the linear layer with dropout, against plain implementations in 64 bits, value by value.

Bounds. An output in bf16 is off by 2^-8 of itself at most. The tensor core cuts its fp32 sum off once per 16 products, so a sum over K
products with magnitudes adding up to S is off by (K / 16 + 2) * 2^-23 * S at most. An activation is off by 2^-19 (1 + |g|) (exp2 and
reciprocal are good to 2^-22, erf to 2^-22 of 1), its slope by 2^-18 (1 + |g|); slopes are below 1.2. Errors of the factors of a product multiply
the other one."""
import math

import philox64
import pytest
import torch
import torch.nn.functional as F

from parameter_server_b200.ops import act8, dropout, gated, linear
from parameter_server_b200.ops import gemm as G

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
# one value, less than a block, one tile and its edges, several tiles, long sums, many tiles with a rest, tiles that are cut
SHAPES = [(1, 1, 1), (2, 8, 8), (3, 33, 17), (1, 2049, 136), (130, 129, 64), (256, 128, 128), (257, 264, 520), (300, 72, 1000), (700, 31, 72), (1025, 1000, 776),
          (16, 2048, 8200), (2600, 1025, 192), (5000, 250, 12300)]


def rand(*shape, seed=0, std=1.0, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * len(shape) + sum(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def near(got, want, slack):
    assert got.shape == want.shape and got.dtype == BF
    off = (got.double() - want).abs()
    worst = (off / (2.0 ** -8 * want.abs() + slack + 1e-30)).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the bound"


def phi(h, act, slope=False):
    if act in (None, "none"):
        return torch.ones_like(h) if slope else h
    if act == "relu":
        return (h > 0).double() if slope else h.clamp(min=0)
    if act == "silu":
        s = torch.sigmoid(h)
        return s * (1 + h * (1 - s)) if slope else h * s
    if act == "gelu":
        cdf = torch.special.ndtr(h)
        return cdf + h * torch.exp(-h * h / 2) / math.sqrt(2 * math.pi) if slope else h * cdf
    a = math.sqrt(2 / math.pi)
    t = torch.tanh(a * (h + 0.044715 * h ** 3))
    return 0.5 * (1 + t) + 0.5 * h * (1 - t * t) * a * (1 + 0.134145 * h * h) if slope else 0.5 * h * (1 + t)


def sum_slack(a, w):
    return (a.shape[1] / 16 + 2) * 2.0 ** -23 * (a.abs() @ w.abs())


def gated64(x, w, b, act):
    """(y, its slack, h, its slack)"""
    x, w = x.double(), w.double()
    h = x @ w.t() + (0 if b is None else b.double())
    sh = sum_slack(x, w.t()) + 2.0 ** -23 * h.abs()
    n = w.shape[0] // 2
    g, u, sg, su = h[:, :n], h[:, n:], sh[:, :n], sh[:, n:]
    p = phi(g, act)
    return p * u, (1.2 * sg + 2.0 ** -19 * (1 + g.abs())) * (u.abs() + su) + p.abs() * su + 2.0 ** -23 * (p * u).abs(), h, sh


def kept_is(kept, h, slack):
    """A checkpoint stands for h: within half a step, and a step no coarser than the rule has it."""
    rows, n = h.shape
    step = torch.ldexp(torch.ones(rows, -(-n // 32), dtype=torch.float64, device="cuda"), kept.e[:, : -(-n // 32)].int() - 127).repeat_interleave(32, 1)[:, :n]
    assert ((act8.act8_unpack(kept, F32).double() - h).abs() <= step / 2 + slack).all()
    top = F.pad(h.abs(), (0, -n % 32)).view(rows, -1, 32).amax(-1).repeat_interleave(32, 1)[:, :n]
    assert (step <= (top + slack.amax()) / 63.7 + 2.0 ** -126).all()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gated_linear(M, N, K, act):
    x, w, b = rand(M, K), rand(2 * N, K, seed=1, std=K ** -0.5), rand(2 * N, seed=2)
    want, slack, h, sh = gated64(x, w, b, act)
    y, pre = gated.gated_linear(x, w, b, act=act, save="bf16")
    near(pre, h, sh)
    near(y, want, slack)
    assert torch.equal(gated.gated_linear(x, w, b.float(), act=act), y)
    y8, (g8, u8) = gated.gated_linear(x, w, b, act=act, save="act8")
    assert torch.equal(y8, y)
    kept_is(g8, h[:, :N], sh[:, :N])
    kept_is(u8, h[:, N:], sh[:, N:])
    want, slack, _, _ = gated64(x, w, None, act)
    near(gated.gated_linear(x, w, act=act), want, slack)
    G.check_gemm_errors()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", SHAPES[:-1] + [(10000, 250, 12300)])
def test_gated_linear_dgrad(M, N, K, act):
    dy, w = rand(M, K), rand(K, N, seed=1, std=K ** -0.5)
    da = dy.double() @ w.double()
    s = sum_slack(dy.double(), w.double())
    h = rand(M, 2 * N, seed=2) * 2
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
def test_gradients_against_differences(act):
    """dh = [da u act'(g) | da act(g)] against y(h + s) - y(h - s), both factors in turn: g and u are products with the identity, y comes in
    bf16 (off by 2^-8 of itself, so a difference over 1/4 by 2^-8 of both over 1/4), and the third derivative's part is under 0.012 |u|."""
    n = 64
    g = torch.linspace(-4, 4, 40 * n, device="cuda").view(40, n).bfloat16()
    u = rand(40, n, seed=3)
    eye = torch.eye(n, device="cuda").bfloat16()
    both = torch.block_diag(eye, eye)
    y = lambda g, u: gated.gated_linear(torch.cat((g, u), 1), both, act=act).double()  # noqa: E731
    dh = gated.gated_linear_dgrad(torch.ones(40, n, device="cuda").bfloat16(), eye, torch.cat((g, u), 1), act=act).double()
    for got, (up, down), apart, curve in (
            (dh[:, :n], (y(g + 0.125, u), y(g - 0.125, u)), (g + 0.125).double() - (g - 0.125).double(), 0.012 * u.double().abs()),
            (dh[:, n:], (y(g, u + 0.125), y(g, u - 0.125)), (u + 0.125).double() - (u - 0.125).double(), 0.0)):
        off = ((up - down) / apart - got).abs()
        if act == "relu":
            off = torch.where(g.double().abs() <= 0.13, torch.zeros_like(off), off)   # the corner
        assert (off <= 2.0 ** -8 * (up.abs() + down.abs()) / apart + 2.0 ** -8 * got.abs() + curve + 1e-6).all(), off.max()


@pytest.mark.parametrize("M,N,K", [(4200, 1100, 136), (4200, 1098, 72), (4200, 1101, 72), (70, 44, 40), (70, 42, 40), (300, 41, 40), (1, 1003, 264)])
def test_results_and_kept_values_on_any_boundary(M, N, K):
    """Rows, and the second half of a row, on multiples of 16, 8, 4 and 2 bytes: bit for bit what padded halves give, and nothing written
    beside them."""
    Np = -(-N // 32) * 32
    pad = lambda w: torch.cat((F.pad(w[:N], (0, 0, 0, Np - N)), F.pad(w[N:], (0, 0, 0, Np - N))))  # noqa: E731
    x, w = rand(M, K), rand(2 * N, K, seed=1)
    y, h = gated.gated_linear(x, w, act="silu", save="bf16")
    wide, hw = gated.gated_linear(x, pad(w), act="silu", save="bf16")
    assert torch.equal(y, wide[:, :N]) and torch.equal(h[:, :N], hw[:, :N]) and torch.equal(h[:, N:], hw[:, Np:Np + N])
    assert y.stride(0) % 8 == 0 and h.stride(0) % 8 == 0
    cols = torch.full((M, N + 3), 7.0, dtype=BF, device="cuda")
    out = cols[:, 1:N + 1]
    assert gated.gated_linear(x, w, act="silu", out=out) is out and torch.equal(out, y)
    assert (cols[:, 0] == 7).all() and (cols[:, N + 1:] == 7).all()
    dy, w2 = rand(M, K, seed=4), rand(K, N, seed=5)
    one = gated.gated_linear_dgrad(dy, w2, h, act="gelu", recompute=True)
    other = gated.gated_linear_dgrad(dy, w2, h.contiguous(), act="gelu", recompute=True)
    dw, aw = gated.gated_linear_dgrad(dy, F.pad(w2, (0, Np - N)), hw, act="gelu", recompute=True)
    assert all(torch.equal(p, q) for p, q in zip(one, other))
    assert torch.equal(one[1], aw[:, :N]) and torch.equal(one[0], torch.cat((dw[:, :N], dw[:, Np:Np + N]), 1))
    G.check_gemm_errors()


def test_strides_dims_and_nothing():
    M, N, K = 200, 136, 72
    wide, w = rand(M, 3 * K), rand(2 * N, K, seed=1, std=0.1)
    for x in (wide[:, K:2 * K], wide[:, 1:K + 1], wide[::2, :K], wide[:, :K].t().contiguous().t(), wide[:1, :K].expand(9, K)):
        assert torch.equal(gated.gated_linear(x, w), gated.gated_linear(x.contiguous(), w))
    odd = rand(2 * N, K + 1, seed=5)[:, 1:]
    assert torch.equal(gated.gated_linear(wide[:, :K], odd), gated.gated_linear(wide[:, :K], odd.contiguous()))
    x3 = wide[:, :K].reshape(4, 50, K)
    y3, h3 = gated.gated_linear(x3, w, save="bf16")
    assert y3.shape == (4, 50, N) and h3.shape == (4, 50, 2 * N) and torch.equal(y3.view(M, N), gated.gated_linear(wide[:, :K], w))
    dy, w2 = rand(4, 50, 24), rand(24, N)
    dh, a = gated.gated_linear_dgrad(dy, w2, h3, recompute=True)
    assert dh.shape == (4, 50, 2 * N) and a.shape == (4, 50, N)
    _, kept = gated.gated_linear(x3, w, save="act8")
    assert gated.gated_linear_dgrad(dy, w2, kept).shape == (4, 50, 2 * N)
    y0, h0 = gated.gated_linear(rand(0, K), w, save="bf16")
    assert y0.shape == (0, N) and gated.gated_linear_dgrad(rand(0, 24), w2, h0).shape == (0, 2 * N)
    assert gated.gated_linear(rand(3, K), rand(0, K)).shape == (3, 0)
    assert torch.equal(gated.gated_linear(wide[:, :K], w.view(2, N, K)), gated.gated_linear(wide[:, :K], w))   # both weights in one tensor
    G.check_gemm_errors()


def test_far_out_and_not_finite():
    n = 16
    g = torch.tensor([0.0, -0.0, 1e4, -1e4, 3e18, -3e18, 3e38, -3e38, 40.0, -40.0, math.inf, math.nan] + [0.5] * 4, device="cuda").bfloat16().view(1, n)
    eye, one = torch.eye(n, device="cuda").bfloat16(), torch.ones(1, n, device="cuda").bfloat16()
    for act in ACTS[1:]:
        dh, a = gated.gated_linear_dgrad(one, eye, torch.cat((g, one), 1), act=act, recompute=True)
        slope, du = dh[:, :n], dh[:, n:]
        assert torch.isnan(slope[0, 11]) and torch.isnan(a[0, 11]) and a[0, 10] == math.inf and du[0, 10] == math.inf
        far = torch.tensor([1, 0, 1, 0, 1, 0, 1, 0], device="cuda").bfloat16()
        assert ((slope[0, 2:10] - far).abs() <= 2.0 ** -50).all() and torch.equal(a[0, :10], du[0, :10])
    x = torch.zeros(4, 64, device="cuda").bfloat16()
    x[0, 0], x[1, 1] = math.nan, math.inf
    w = rand(80, 64)
    y, (g8, u8) = gated.gated_linear(x, w, act="gelu", save="act8")
    v = act8.act8_unpack(g8), act8.act8_unpack(u8)
    assert torch.isnan(y[0]).all() and (y[2:] == 0).all() and all(torch.isnan(k[:2]).all() and (k[2:] == 0).all() for k in v)


def test_rows_of_w_behind_the_gates_do_not_reach_its_checkpoint():
    """A gate of 40 rows ends inside a block of 32 and inside a tile; the rows behind it are large, or not finite."""
    x, w = rand(300, 64), rand(80, 64, seed=1)
    for rows in (300, 5):
        _, (g8, _) = gated.gated_linear(x[:rows], w, save="act8")
        for huge in (1e30, math.nan):
            v = w.clone()
            v[40:] = huge
            _, (k8, _) = gated.gated_linear(x[:rows], v, save="act8")
            assert torch.equal(act8.act8_unpack(k8), act8.act8_unpack(g8))


def test_repeats_bit_for_bit_on_any_stream_and_in_a_graph():
    x, w = rand(5000, 12300), rand(500, 12300, seed=1, std=0.01)           # cut along the contraction
    dy, w2, h = rand(16, 1024), rand(1024, 512, seed=2, std=0.03), rand(16, 1024, seed=3)
    y, dh = gated.gated_linear(x, w), gated.gated_linear_dgrad(dy, w2, h)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys = [gated.gated_linear(x, w) for _ in range(3)]
        ds = [gated.gated_linear_dgrad(dy, w2, h) for _ in range(3)]
    more = [gated.gated_linear(x, w) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, v) for v in ys + more) and all(torch.equal(dh, v) for v in ds)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append((gated.gated_linear(x, w), gated.gated_linear_dgrad(dy, w2, h)))
    for _ in range(2):
        for graph, (gy, gd) in zip(graphs, outs):
            gy.zero_(), gd.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(gy, y) and torch.equal(gd, dh)
    G.check_gemm_errors()


def test_overlapping_launches_keep_their_order():
    """A training step of the gated layer over and over, with and without a wait between its launches."""
    D, H = 512, 700

    def chain(tokens, wait):
        w1, w2, b1 = rand(2 * H, D, std=0.05), rand(D, H, std=0.05, seed=1), rand(2 * H, seed=2)
        x, dw, db = rand(tokens, D, seed=5), torch.zeros(2 * H, D, device="cuda"), torch.zeros(2 * H, device="cuda")
        stop = torch.cuda.synchronize if wait else (lambda: None)
        for step in range(8):
            a, h = gated.gated_linear(x, w1, b1, save="bf16" if step % 2 else "act8"); stop()
            y = linear.linear_act(a, w2, residual=x, dropout=(0.1, 7, step)); stop()
            dz = dropout.dropout_backward(y, 0.1, 7, step); stop()
            dh, a = gated.gated_linear_dgrad(dz, w2, h, recompute=True); stop()
            linear.linear_bias_grad(dh, out=db, accumulate=True); stop()
            G.gemm(dh, x, a_mn=True, b_mn=True, out=dw, accumulate=True); stop()
            dx = linear.linear_act_dgrad(dh, w1, None); stop()
            x = dropout.dropout(dx, 0.5, 3, step, residual=x, out=dx); stop()
            x = act8.act8_unpack(act8.act8_pack(x)); stop()
            x = x / x.abs().amax()   # (a step's result grows with the third power of its input)
        return x, dw, db

    for tokens in (8, 136, 1024):
        one, other = chain(tokens, True), chain(tokens, False)
        assert all(torch.equal(p, q) for p, q in zip(one, other)) and all(torch.isfinite(p).all() for p in one)
    G.check_gemm_errors()


def test_a_limit_of_ctas_and_a_wait_that_has_no_time():
    x, w = rand(300, 512), rand(520, 512, seed=1)
    want = gated.gated_linear(x, w)
    from parameter_server_b200._lib import C
    C.gemm_set_cta_limit(16)
    try:
        near(gated.gated_linear(x, w), *gated64(x, w, None, "silu")[:2])
    finally:
        C.gemm_set_cta_limit(0)
    assert torch.equal(gated.gated_linear(x, w), want)
    G.check_gemm_errors()


# ---- dropout in the epilogue --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (3, 33, 17), (130, 129, 64), (257, 264, 520), (1025, 1000, 776), (16, 2048, 8200), (2600, 1025, 192), (5000, 500, 12300), (128, 6, 40)])
def test_linear_with_dropout(M, N, K, act):
    x, w, b, r = rand(M, K), rand(N, K, seed=1, std=K ** -0.5), rand(N, seed=2), rand(M, N, seed=3)
    seed, offset, p = 0xFEDCBA9876543210, (1 << 35) + 9, 0.35
    mask = torch.from_numpy(philox64.kept(M, N, p, seed, offset)).cuda()
    h = x.double() @ w.double().t() + b.double()
    v = phi(h, act)
    slack = philox64.grown(p) * (1.2 * (sum_slack(x.double(), w.double().t()) + 2.0 ** -23 * h.abs()) + 2.0 ** -19 * (1 + h.abs()))
    want, slack = torch.where(mask, philox64.grown(p) * v, 0.0), torch.where(mask, slack, 0.0)
    y, pre = linear.linear_act(x, w, b, act=act, residual=r, save="bf16", dropout=(p, seed, offset))
    near(y, want + r.double(), slack + 2.0 ** -22 * (want.abs() + r.double().abs()))
    assert torch.equal(pre, linear.linear_act(x, w, b, act=act, save="bf16")[1])
    alone = linear.linear_act(x, w, b, act=act, dropout=(p, torch.tensor([seed - (1 << 64)], device="cuda"), offset))
    near(alone, want, slack + 2.0 ** -22 * want.abs())
    assert torch.equal(alone != 0, mask & (alone != 0)) and (alone[~mask] == 0).all()
    assert torch.equal(linear.linear_act(x, w, b, act=act, residual=r, dropout=(0.0, seed, offset)), linear.linear_act(x, w, b, act=act, residual=r))
    # the mask is that of dropout itself, and its backward pass
    assert (dropout.dropout_backward(torch.ones(M, N, dtype=BF, device="cuda"), p, seed, offset) != 0).equal(mask)
    G.check_gemm_errors()
