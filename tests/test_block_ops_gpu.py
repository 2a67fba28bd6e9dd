"""Layer norm, fused linear layers and 8-bit checkpoints against plain implementations in 64 bits.

Bounds: an output rounded to bf16 is off by 2^-8 of itself at most, to fp32 by 2^-24. The tensor core cuts its fp32 sum off once per 16
products, so a sum over K products with magnitudes adding up to S is off by (K / 16 + 2) * 2^-23 * S at most; in the weight gradient
such a chain ends after 512 tokens and the chains are added with one rounding each. Everything is compared element by element."""
import math

import pytest
import torch
import torch.nn.functional as F

from parameter_server_b200._lib import C
from parameter_server_b200.ops import act8, linear, norm
from parameter_server_b200.ops import gemm as G

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
ULP = {BF: 2.0 ** -8, F32: 2.0 ** -23}   # one rounding (fp32: and one ahead of it)


def rand(*shape, seed=0, std=1.0, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * len(shape) + sum(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def near(got, want, slack=0.0):
    """Element by element within one rounding of `want` (64 bits) and `slack`."""
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    bound = ULP[got.dtype] * want.abs() + slack + 1e-30
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the bound"


# ---- the 8-bit format --------------------------------------------------------------------------------------------------

def power(e):
    """2^(e-127), exactly (torch.pow on the GPU is not)."""
    return torch.ldexp(torch.ones_like(e), (e - 127).int())


def quantise(x):
    """(q, exponent byte) of rows, by the definition: the smallest step 2^(e-127) at which the block's largest rounds to 127 or less."""
    x = x.double()
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = torch.zeros(rows, blocks * 32, dtype=torch.float64, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, blocks, 32)
    top = v.abs().amax(-1)
    fine = torch.isfinite(v).all(-1)
    e = torch.full_like(top, 1.0)
    for k in range(1, 250):
        e = torch.where(top / 2.0 ** (k - 127) >= 127.5, torch.full_like(e, k + 1.0), e)
    q = torch.round(v / power(e).unsqueeze(-1))
    q = torch.where(fine.unsqueeze(-1), q, torch.zeros_like(q))
    e = torch.where(fine, e, torch.full_like(e, 255.0))
    return q.view(rows, -1)[:, :cols], e


def stands_for(q, e):
    step = torch.where(e == 255, torch.full_like(e, math.nan), power(e))
    return q * step.repeat_interleave(32, 1)[:, : q.shape[1]]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (5, 32), (7, 33), (2, 257), (64, 1000), (33, 2048), (4, 9000)])
def test_pack_is_the_definition(rows, cols, dtype):
    x = rand(rows, cols, dtype=dtype) * torch.exp(4 * rand(rows, 1, dtype=F32, seed=1)).to(dtype)
    a = act8.act8_pack(x)
    q, e = quantise(x)
    assert torch.equal(a.q[:, :cols].double(), q) and torch.equal(a.e[:, : e.shape[1]].double(), e)
    for out in (BF, F32):
        assert torch.equal(act8.act8_unpack(a, out).double(), stands_for(q, e))


def test_pack_at_the_edges():
    x = torch.zeros(9, 64, device="cuda")
    x[1, 3] = 127.4999                      # stays at step 1
    x[2, 3] = 127.5                         # would round to 128: step 2
    x[3, :2] = torch.tensor([2.0 ** -140, -(2.0 ** -133)])
    x[4, 5] = math.inf
    x[5, 40] = math.nan
    x[6, :] = -1.5
    x[7, 0], x[7, 1] = 3.0e38, -1.0e38
    x[8, 0], x[8, 1] = 127.0, 0.5           # a tie goes to the even number
    a = act8.act8_pack(x)
    q, e = quantise(x)
    assert torch.equal(a.q[:, :64].double(), q) and torch.equal(a.e[:, :2].double(), e)
    v = act8.act8_unpack(a, F32)
    assert torch.isnan(v[4, :32]).all() and (v[4, 32:] == 0).all() and torch.isnan(v[5, 32:]).all() and (v[5, :32] == 0).all()
    assert v[1, 3] == 127 and v[2, 3] == 128 and v[8, 1] == 0 and (v[6] == -1.5).all()
    assert (v[7, 0] - 3.0e38).abs() <= 3.0e38 / 127


def test_pack_reads_strided_and_shifted_rows():
    base = rand(40, 200)
    for x in (base[:, 3:180], base[::2, 8:136], base.t()[16:80], base[:, 5:6]):
        q, e = quantise(x)
        a = act8.act8_pack(x)
        assert torch.equal(act8.act8_unpack(a).double(), stands_for(q, e))
    x = rand(2, 3, 64)
    assert act8.act8_pack(x).shape == (6, 64)
    assert act8.act8_pack(rand(0, 64)).shape == (0, 64)


# ---- layer norm --------------------------------------------------------------------------------------------------------

EPS = 1e-5


def norm64(x, g, b, eps=EPS):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = ((x - mean).square().mean(1, keepdim=True) + eps) ** -0.5
    xhat = (x - mean) * rstd
    y = xhat * (1.0 if g is None else g.double()) + (0.0 if b is None else b.double())
    return y, mean.squeeze(1), rstd.squeeze(1), xhat


def norm64_grads(dy, xhat, rstd, g, join):
    p = dy.double() * (1.0 if g is None else g.double())
    dx = rstd[:, None] * (p - p.mean(1, keepdim=True) - xhat * (p * xhat).mean(1, keepdim=True))
    return (dx if join is None else dx + join.double()), (dy.double() * xhat).sum(0), dy.double().sum(0)


def norm_slack(x, xhat):
    """Error of a normalised value: x and the mean enter with 2^-24 of the largest |x| over the row's deviation, the sums' roundings
    (a few per value, in a tree) stay below 2^-20 of the values."""
    dev = (x.double().var(1, unbiased=False, keepdim=True) + EPS).sqrt()
    return 2.0 ** -22 * x.double().abs().amax(1, keepdim=True) / dev + 2.0 ** -20 * (1 + xhat.abs())


NORM_SHAPES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 100), (700, 96), (17, 1001), (640, 2048), (5, 2049), (3, 8192), (2, 8200), (2, 20000), (2, 33000)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,d", NORM_SHAPES)
def test_layer_norm_forward(rows, d, dtype):
    x = rand(rows, d, dtype=dtype) * 3 + 1
    g, b = rand(d, seed=1, dtype=dtype), rand(d, seed=2, dtype=dtype)
    y, mean, rstd = norm.layer_norm(x, g, b, EPS)
    ry, rm, rr, xhat = norm64(x, g, b)
    slack = norm_slack(x, xhat) * (1 + g.double().abs())
    near(y, ry, slack)
    near(mean, rm, 2.0 ** -22 * x.double().abs().amax(1))
    near(rstd, rr, 2.0 ** -20 * rr)
    y8, x8, rstd8 = norm.layer_norm_act8(x, g, b, EPS)
    assert torch.equal(y8, y) and torch.equal(rstd8, rstd)
    # half a step of the block, from the normalised value itself
    step = power(x8.e[:, : -(-d // 32)].double()).repeat_interleave(32, 1)[:, :d]
    assert ((act8.act8_unpack(x8, F32).double() - xhat).abs() <= step / 2 + norm_slack(x, xhat)).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("join", [False, True])
@pytest.mark.parametrize("rows,d", NORM_SHAPES)
def test_layer_norm_backward(rows, d, join, dtype):
    x = rand(rows, d, dtype=dtype) * 3 + 1
    g = rand(d, seed=1, dtype=dtype)
    dy = rand(rows, d, seed=3, dtype=dtype)
    j = rand(rows, d, seed=4, dtype=dtype) if join else None
    y, mean, rstd = norm.layer_norm(x, g, None, EPS)
    dx, dw, db = norm.layer_norm_backward(dy, x, g, mean, rstd, residual_grad=j)
    xhat = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    rx, rw, rb = norm64_grads(dy, xhat, rstd.double(), g, j)
    p = (dy.double() * g.double()).abs()
    # two row sums of d terms and one product each: roundings of 2^-24 against what was added
    slack = rstd.double()[:, None] * 2.0 ** -20 * (p + p.mean(1, keepdim=True) + xhat.abs() * (p * xhat.abs()).mean(1, keepdim=True)) + 2.0 ** -24 * rx.abs()
    near(dx, rx, slack)
    near(dw, rw, 2.0 ** -20 * (dy.double() * xhat).abs().sum(0))
    near(db, rb, 2.0 ** -20 * dy.double().abs().sum(0))
    # from the checkpoint: the same formula on the values that it stands for
    _, x8, rstd8 = norm.layer_norm_act8(x, g, None, EPS)
    kept = act8.act8_unpack(x8, F32).double()
    dx, dw, db8 = norm.layer_norm_act8_backward(dy, x8, g, rstd8, residual_grad=j)
    rx, rw, rb = norm64_grads(dy, kept, rstd8.double(), g, j)
    slack = rstd.double()[:, None] * 2.0 ** -20 * (p + p.mean(1, keepdim=True) + kept.abs() * (p * kept.abs()).mean(1, keepdim=True)) + 2.0 ** -24 * rx.abs()
    near(dx, rx, slack)
    near(dw, rw, 2.0 ** -20 * (dy.double() * kept).abs().sum(0))
    near(db8, rb, 2.0 ** -20 * dy.double().abs().sum(0))


def test_layer_norm_backward_against_differences():
    rows, d = 6, 300
    x, g, b, dy, v = (rand(rows, d, dtype=F32), rand(d, seed=1, dtype=F32), rand(d, seed=2, dtype=F32), rand(rows, d, seed=3, dtype=F32),
                      rand(rows, d, seed=4, dtype=F32))
    _, mean, rstd = norm.layer_norm(x, g, b)
    dx, dw, db = norm.layer_norm_backward(dy, x, g, mean, rstd)
    loss = lambda x, g, b: (norm.layer_norm(x, g, b)[0].double() * dy.double()).sum()  # noqa: E731
    h = 2.0 ** -7   # the forward pass is off by 2^-24 of its values (their sum's size is sqrt(rows d) = 42); third derivatives are of order 1
    for slope, plus, minus in (((dx.double() * v.double()).sum(), loss(x + h * v, g, b), loss(x - h * v, g, b)),
                               ((dw.double() * v[0].double()).sum(), loss(x, g + h * v[0], b), loss(x, g - h * v[0], b)),
                               ((db.double() * v[0].double()).sum(), loss(x, g, b + h * v[0]), loss(x, g, b - h * v[0]))):
        assert abs(((plus - minus) / (2 * h) - slope).item()) < 0.02 + 2e-3 * abs(slope.item())


def test_layer_norm_special_rows():
    x = rand(6, 256, dtype=F32)
    x[0] = 4.0                          # no deviation: rstd = eps^-1/2, the row is 0
    x[1, 3], x[2, 7] = math.nan, math.inf
    x[3] = x[3] + 4096.0                # far from zero: the distances are taken from the mean
    g, b = rand(256, seed=1, dtype=F32), rand(256, seed=2, dtype=F32)
    y, mean, rstd = norm.layer_norm(x, g, b)
    assert torch.allclose(y[0], b) and abs(rstd[0].item() * EPS ** 0.5 - 1) < 1e-5
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and torch.isfinite(y[3:]).all()
    ry, _, _, xhat = norm64(x[3:], g, b)
    near(y[3:], ry, norm_slack(x[3:], xhat) * (1 + g.double().abs()))
    _, x8, _ = norm.layer_norm_act8(x, g, b)
    v = act8.act8_unpack(x8)
    assert torch.isnan(v[1]).all() and (v[0] == 0).all()
    dx, dw, db = norm.layer_norm_backward(torch.ones_like(x), x, g, mean, rstd)
    assert torch.isnan(dx[1]).all() and torch.isfinite(dx[3:]).all() and torch.isnan(dw[3]) and torch.isfinite(db).all()


def test_layer_norm_strides_dims_and_missing_parts():
    base = rand(2, 50, 3, 64)
    x = base[:, :, 1]                              # rows 192 apart
    y, mean, rstd = norm.layer_norm(x)
    ry, _, _, xhat = norm64(x.reshape(-1, 64), None, None)
    near(y.reshape(-1, 64), ry, norm_slack(x.reshape(-1, 64), xhat))
    assert y.shape == x.shape and mean.shape == (100,)
    dy = rand(2, 50, 64, seed=5)
    dx, dw, db = norm.layer_norm_backward(dy, x, None, mean, rstd)
    assert dx.shape == x.shape
    dx2, dw2, _ = norm.layer_norm_backward(dy.reshape(-1, 64), x.reshape(-1, 64).contiguous(), None, mean, rstd)
    assert torch.equal(dx.reshape(-1, 64), dx2) and torch.equal(dw, dw2)
    for v in (rand(40, 200)[:, 1:130], rand(40, 129).t()):   # rows that no 16-byte access fits, columns for rows
        y, _, _ = norm.layer_norm(v)
        ry, _, _, xhat = norm64(v, None, None)
        near(y, ry, norm_slack(v, xhat))
    y, mean, rstd = norm.layer_norm(rand(0, 64))
    assert y.shape == (0, 64) and mean.numel() == 0
    dx, dw, db = norm.layer_norm_backward(rand(0, 64), rand(0, 64), None, mean, rstd)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()


def test_layer_norm_gradients_accumulate_and_repeat_bit_for_bit():
    x, dy, g = rand(3000, 512), rand(3000, 512, seed=1), rand(512, seed=2)
    _, mean, rstd = norm.layer_norm(x, g)
    first = norm.layer_norm_backward(dy, x, g, mean, rstd)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, norm.layer_norm_backward(dy, x, g, mean, rstd)))
    w, b = torch.full((512,), 2.0, device="cuda"), torch.full((512,), -1.0, device="cuda")
    _, w2, b2 = norm.layer_norm_backward(dy, x, g, mean, rstd, weight_grad=w, bias_grad=b, accumulate=True)
    assert w2 is w and b2 is b and torch.equal(w, first[1] + 2) and torch.equal(b, first[2] - 1)


# ---- fused linear ------------------------------------------------------------------------------------------------------

def phi(h, act, slope=False):
    if act in (None, "none"):
        return torch.ones_like(h) if slope else h
    if act == "relu":
        return (h > 0).double() if slope else h.clamp(min=0)
    if act == "silu":
        s = torch.sigmoid(h)
        return s * (1 + h * (1 - s)) if slope else h * s
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(h / math.sqrt(2)))
        return cdf + h * torch.exp(-h * h / 2) / math.sqrt(2 * math.pi) if slope else h * cdf
    a = math.sqrt(2 / math.pi)
    t = torch.tanh(a * (h + 0.044715 * h ** 3))
    return 0.5 * (1 + t) + 0.5 * h * (1 - t * t) * a * (1 + 0.134145 * h * h) if slope else 0.5 * h * (1 + t)


def sum_slack(a, w):
    """a [M, K], w [K, N] in 64 bits: how far the tensor core's sum may be off."""
    return (a.shape[1] / 16 + 2) * 2.0 ** -23 * (a.abs() @ w.abs())


ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
# one value, less than a block, one tile and its edges, several tiles, many tiles with a rest, long sums that are cut
LINEAR_SHAPES = [(1, 1, 1), (2, 8, 8), (3, 33, 17), (130, 129, 64), (256, 256, 128), (257, 264, 520), (300, 72, 1000), (1025, 1000, 776), (16, 2048, 8200), (2600, 2048, 192)]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", LINEAR_SHAPES)
def test_linear_act(M, N, K, act):
    x, w, b, r = rand(M, K), rand(N, K, seed=1, std=K ** -0.5), rand(N, seed=2), rand(M, N, seed=3)
    h = x.double() @ w.double().t() + b.double()
    slack = sum_slack(x.double(), w.double().t())
    soft = 2.0 ** -19 * (1 + h.abs())   # exp2 and reciprocal are good to 2^-22, erf to 2^-22 of 1
    y, pre = linear.linear_act(x, w, b, act=act, residual=r, save="bf16")
    near(pre, h, slack)
    near(y, phi(h, act) + r.double(), 1.2 * slack + soft + 2.0 ** -23 * r.double().abs())
    near(linear.linear_act(x, w, act=act), phi(h - b.double(), act), 1.2 * slack + soft + 2.0 ** -20 * b.double().abs())
    near(linear.linear_act(x, w, b.float(), act=act), phi(h, act), 1.2 * slack + soft)
    y8, kept = linear.linear_act(x, w, b, act=act, residual=r, save="act8")
    assert torch.equal(y8, y)
    step = power(kept.e[:, : -(-N // 32)].double()).repeat_interleave(32, 1)[:, :N]
    v = act8.act8_unpack(kept, F32).double()
    assert ((v - h).abs() <= step / 2 + slack + 2.0 ** -22 * h.abs()).all()
    top = torch.nn.functional.pad(h.abs(), (0, -N % 32)).view(M, -1, 32).amax(-1).repeat_interleave(32, 1)[:, :N]
    assert (step <= (top + slack.amax()) / 63.7 + 2.0 ** -126).all()   # no coarser than the rule has it
    G.check_gemm_errors()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", LINEAR_SHAPES)
def test_linear_act_dgrad(M, N, K, act):
    dy, w = rand(M, K), rand(K, N, seed=1, std=K ** -0.5)
    z = dy.double() @ w.double()
    slack = sum_slack(dy.double(), w.double())
    h = rand(M, N, seed=2) * 3
    for kept, value in ((h, h.double()), (act8.act8_pack(h), act8.act8_unpack(act8.act8_pack(h), F32).double())):
        dh, a = linear.linear_act_dgrad(dy, w, kept, act=act, recompute=True)
        near(dh, z * phi(value, act, slope=True), 1.2 * slack + 2.0 ** -18 * z.abs() * (1 + value.abs()))
        near(a, phi(value, act), 2.0 ** -19 * (1 + value.abs()))
        assert torch.equal(linear.linear_act_dgrad(dy, w, kept, act=act), dh)
    if act == "none":
        near(linear.linear_act_dgrad(dy, w, None), z, slack)
    G.check_gemm_errors()


@pytest.mark.parametrize("act", ACTS)
def test_slopes_against_differences(act):
    """h goes through as its own product with the identity; y comes in bf16, off by 2^-8 of itself, so a difference over 1/4 is off by
    2^-8 of both over 1/4 and by the third derivative's part, under 0.012; the slope itself by its rounding."""
    n = 64
    h = torch.linspace(-4, 4, 40 * n, device="cuda").view(40, n).bfloat16()
    eye = torch.eye(n, device="cuda").bfloat16()
    up, down = (linear.linear_act(h + s, eye, act=act).double() for s in (0.125, -0.125))
    apart = (h + 0.125).double() - (h - 0.125).double()   # as bf16 has them
    slope = linear.linear_act_dgrad(torch.ones(40, n, device="cuda").bfloat16(), eye, h, act=act).double()
    # (dy of ones times the identity is 1 in every place)
    off = ((up - down) / apart - slope).abs()
    if act == "relu":
        off = torch.where(h.double().abs() <= 0.13, torch.zeros_like(off), off)   # the corner
    assert (off <= 2.0 ** -8 * (up.abs() + down.abs()) / apart + 2.0 ** -8 * slope.abs() + 0.012).all(), off.max()


def test_activations_far_out_and_not_finite():
    h = torch.tensor([0.0, -0.0, 1e4, -1e4, 3e18, -3e18, 3e38, -3e38, 40.0, -40.0, math.inf, math.nan] + [0.5] * 4, device="cuda").bfloat16().view(1, 16)
    eye = torch.eye(16, device="cuda").bfloat16()
    one = torch.ones(1, 16, device="cuda").bfloat16()
    for act in ACTS[1:]:
        slope, a = linear.linear_act_dgrad(one, eye, h, act=act, recompute=True)
        assert torch.isnan(slope[0, 11]) and torch.isnan(a[0, 11]) and a[0, 10] == math.inf
        far = torch.tensor([1, 0, 1, 0, 1, 0, 1, 0], device="cuda").bfloat16()
        # silu(-40) = -40 / (1 + e^40) and its slope are not 0 but about 2^-52; all others have underflowed
        assert ((slope[0, 2:10] - far).abs() <= 2.0 ** -50).all(), (act, slope)
        assert torch.equal(a[0, 2:9], torch.where(far > 0, h[0, 2:10], torch.zeros_like(far))[:7]) and a[0, 9].abs() <= 2.0 ** -50, (act, a)
    x = torch.zeros(3, 64, device="cuda").bfloat16()
    x[0, 0], x[1, 1] = math.nan, math.inf
    w = rand(40, 64)
    y, kept = linear.linear_act(x, w, act="gelu", save="act8")
    v = act8.act8_unpack(kept)
    assert torch.isnan(y[0]).all() and torch.isnan(v[0]).all() and torch.isnan(v[1]).all() and (y[2] == 0).all() and (v[2] == 0).all()


def test_linear_strides_alignment_and_places():
    M, N, K = 200, 136, 72
    wide = rand(M, 3 * K)
    w, b, r = rand(N, K, seed=1), rand(N, seed=2), rand(M, N, seed=3)
    for x in (wide[:, K:2 * K], wide[:, 1:K + 1], wide[::2, :K], wide[:, :K].t().contiguous().t()):
        rr = r[: x.shape[0]]
        got = linear.linear_act(x, w, b, residual=rr)
        near(got, x.double() @ w.double().t() + b.double() + rr.double(), sum_slack(x.double(), w.double().t()) + 2.0 ** -22)
    x = wide[:, :K]
    want = linear.linear_act(x, w, b, residual=r)
    out = torch.zeros(M, N + 5, device="cuda").bfloat16()          # rows that no 16-byte store fits
    assert linear.linear_act(x, w, b, residual=r, out=out[:, 2:N + 2]).data_ptr() == out[:, 2:].data_ptr()
    assert torch.equal(out[:, 2:N + 2], want) and (out[:, :2] == 0).all() and (out[:, N + 2:] == 0).all()
    res = r.clone()
    assert torch.equal(linear.linear_act(x, w, b, residual=res, out=res), want) and torch.equal(res, want)   # in place
    x3 = x.reshape(4, 50, K)
    y3, h3 = linear.linear_act(x3, w, b, residual=r.view(4, 50, N), save="bf16")
    assert y3.shape == (4, 50, N) and torch.equal(y3.view(M, N), want)
    assert linear.linear_act_dgrad(rand(4, 50, 24), rand(24, N), h3, act="silu").shape == (4, 50, N)
    odd = rand(N, K + 1, seed=5)[:, 1:]                             # an unaligned weight
    near(linear.linear_act(x, odd), x.double() @ odd.double().t(), sum_slack(x.double(), odd.double().t()))
    assert linear.linear_act(rand(0, K), w).shape == (0, N)
    G.check_gemm_errors()


def test_cut_tiles_repeat_bit_for_bit_and_on_another_stream():
    M, N, K = 16, 2048, 16384                                       # fewer tiles than pairs, long sums: cut along K
    x, w = rand(M, K), rand(N, K, seed=1, std=K ** -0.5)
    y = linear.linear_act(x, w, act="gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys = [linear.linear_act(x, w, act="gelu") for _ in range(4)]
    more = [linear.linear_act(x, w, act="gelu") for _ in range(4)]  # beside it, with its own scratch
    torch.cuda.synchronize()
    assert all(torch.equal(y, v) for v in ys + more)
    near(y, phi(x.double() @ w.double().t(), "gelu"), 1.2 * sum_slack(x.double(), w.double().t()) + 2.0 ** -18)
    G.check_gemm_errors()


def test_operators_in_a_captured_graph():
    x, w, dy = rand(64, 16384), rand(512, 16384, seed=1, std=2.0 ** -7), rand(4096, 512, seed=2)
    x8 = act8.act8_pack(rand(4096, 256, seed=3))
    y, dw = linear.linear_act(x, w), act8.act8_wgrad(dy, x8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gy, gw = linear.linear_act(x, w), act8.act8_wgrad(dy, x8)
    for _ in range(3):
        gy.zero_(), gw.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(gy, y) and torch.equal(gw, dw)
    G.check_gemm_errors()


# ---- gradients of weight and bias --------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("M,N", [(1, 1), (3, 130), (777, 33), (5000, 1024), (64, 4099)])
def test_linear_bias_grad(M, N, dtype):
    dy = rand(M, N, dtype=dtype)
    want = dy.double().sum(0)
    got = linear.linear_bias_grad(dy)
    near(got, want, 2.0 ** -21 * dy.double().abs().sum(0))
    assert torch.equal(got, linear.linear_bias_grad(dy))
    out = torch.full((N,), 3.0, device="cuda")
    assert torch.equal(linear.linear_bias_grad(dy, out=out, accumulate=True), got + 3.0) and (linear.linear_bias_grad(dy[:0]) == 0).all()


# one value, less than a stage of tokens, tile edges, several tiles, tokens cut into runs, wide enough to be unpacked first
@pytest.mark.parametrize("T,N,K", [(1, 1, 1), (3, 33, 17), (64, 256, 256), (63, 257, 264), (300, 72, 1000), (130, 128, 64), (5000, 130, 40), (9000, 512, 256), (200, 2056, 4100)])
@pytest.mark.parametrize("form", ["plain", "norm", "accumulate"])
def test_act8_wgrad(T, N, K, form):
    dy = rand(T, N)
    x8 = act8.act8_pack(rand(T, K, seed=1) * 2)
    x = act8.act8_unpack(x8, F32).double()
    size = dy.double().abs().t() @ x.abs()
    slack = (34 * 2.0 ** -23 + (T / 512 + 8) * 2.0 ** -24) * size
    if form == "norm":
        g, b, s = rand(K, seed=2), rand(K, seed=3), linear.linear_bias_grad(dy)
        got = act8.act8_wgrad(dy, x8, weight=g, bias=b, dy_sum=s)
        want = dy.double().t() @ (x * g.double() + b.double())
        slack = slack * g.double().abs() + 2.0 ** -20 * dy.double().abs().sum(0)[:, None] * b.double().abs() + 2.0 ** -22 * want.abs()
    elif form == "accumulate":
        base = rand(N, K, seed=4, dtype=F32)
        out = base.clone()
        got = act8.act8_wgrad(dy, x8, out=out, accumulate=True)
        assert got is out
        want = base.double() + dy.double().t() @ x
        slack = slack + 2.0 ** -23 * base.double().abs()
    else:
        got = act8.act8_wgrad(dy, x8)
        want = dy.double().t() @ x
        assert torch.equal(got, act8.act8_wgrad(dy, x8))
    near(got, want, slack)
    G.check_gemm_errors()


def test_act8_wgrad_every_token_lands_where_it_belongs():
    """With dy a permutation of the unit vectors dw is x itself: a stale or misplaced tile of the checkpoint shows as it is."""
    T, K = 4096, 1024
    order = torch.randperm(T, generator=torch.Generator().manual_seed(3)).cuda()
    dy = torch.zeros(T, T, device="cuda").bfloat16()
    dy[torch.arange(T, device="cuda"), order] = 1
    for k in (K, 1536):                                             # converted tile by tile, and unpacked first (128 tiles and more)
        x8 = act8.act8_pack(rand(T, 2 * k, seed=k))
        x = act8.act8_unpack(x8, F32)
        for _ in range(3):
            assert torch.equal(act8.act8_wgrad(dy, x8)[order], x)
    G.check_gemm_errors()


def test_act8_wgrad_converted_tiles_are_the_right_ones():
    """The same for a layer of few outputs, whose checkpoint is converted tile by tile: some tokens' rows of x at a time."""
    T, N, K = 4096, 1536, 2048
    x8 = act8.act8_pack(rand(T, K, seed=9))
    x = act8.act8_unpack(x8, F32)
    for part in range(4):
        tokens = torch.randperm(T, generator=torch.Generator().manual_seed(part))[:N].cuda()
        dy = torch.zeros(T, N, device="cuda").bfloat16()
        dy[tokens, torch.arange(N, device="cuda")] = 1
        for _ in range(3):
            assert torch.equal(act8.act8_wgrad(dy, x8), x[tokens])
    G.check_gemm_errors()


def test_act8_wgrad_strides_not_finite_and_large_values():
    T, N, K = 300, 96, 160
    wide = rand(T, 3 * N)
    x = rand(T, K, seed=1)
    x[7, 40] = math.nan
    x8 = act8.act8_pack(x)
    v = act8.act8_unpack(x8, F32)
    for dy in (wide[:, N:2 * N], wide[:, 3:N + 3]):
        got = act8.act8_wgrad(dy, x8)
        assert torch.isnan(got[:, 32:64]).all()
        fine = torch.ones(K, dtype=torch.bool, device="cuda")
        fine[32:64] = False
        a, b = dy.double(), v[:, fine].double()
        near(got[:, fine], a.t() @ b, (34 * 2.0 ** -23 + 9 * 2.0 ** -24) * (a.abs().t() @ b.abs()))
    out = torch.zeros(N, K + 3, device="cuda")
    act8.act8_wgrad(wide[:, :N], x8, out=out[:, 1:K + 1])
    assert torch.equal(out[:, 1:33], act8.act8_wgrad(wide[:, :N], x8)[:, :32]) and (out[:, 0] == 0).all() and (out[:, K + 1:] == 0).all()
    big = act8.act8_pack((rand(64, 64, seed=2) * 2.0 ** 110).float())
    got = act8.act8_wgrad(rand(64, 64) * 2.0 ** -100, big)
    a, b = (rand(64, 64) * 2.0 ** -100).double(), act8.act8_unpack(big, F32).double()
    near(got, a.t() @ b, (34 * 2.0 ** -23 + 9 * 2.0 ** -24) * (a.abs().t() @ b.abs()))
    assert (act8.act8_wgrad(rand(0, 8), act8.act8_pack(rand(0, 40))) == 0).all()


# ---- more than 2^31 values ---------------------------------------------------------------------------------------------

def test_offsets_past_32_bits():
    if torch.cuda.get_device_properties(0).total_memory < 60e9:
        pytest.skip("needs 30 GB")
    rows, d = (1 << 31) // 4096 + 300, 4096
    tail = slice(rows - 4, rows)
    x = torch.zeros(rows, d, dtype=BF, device="cuda")
    x[tail] = rand(4, d)
    y, mean, rstd = norm.layer_norm(x)
    near(y[tail], norm64(x[tail], None, None)[0], norm_slack(x[tail], norm64(x[tail], None, None)[3]))
    kept = act8.act8_pack(x)
    assert torch.equal(act8.act8_unpack(act8.Act8(kept.q[tail], kept.e[tail], d)).double(), stands_for(*quantise(x[tail])))
    w = rand(d, 64, seed=1)
    dy = torch.zeros(rows, 64, dtype=BF, device="cuda")
    dy[tail] = rand(4, 64, seed=2)
    z = dy[tail].double() @ w.double().t()
    near(linear.linear_act(dy, w, residual=y, out=y)[tail], z + norm64(x[tail], None, None)[0].bfloat16().double(), sum_slack(dy[tail].double(), w.double().t()) + 0.04)
    del y
    dw = act8.act8_wgrad(dy, kept)
    v = stands_for(*quantise(x[tail]))
    a = dy[tail].double()
    near(dw, a.t() @ v, 34 * 2.0 ** -23 * (a.abs().t() @ v.abs()))
    G.check_gemm_errors()


def test_overlapping_launches_keep_their_order():
    """Launches that may start beside their predecessor's tail give what they give one at a time: a chain in which every one reads
    what the one before wrote, over buffers that are written again and again, with and without a wait between them."""
    T, D, H = 1024, 512, 1024
    w1, w2, b1, g, b = rand(H, D, std=0.05), rand(D, H, std=0.05, seed=1), rand(H, seed=2), rand(D, seed=3), rand(D, seed=4)

    def chain(tokens, wait):
        x, dw, db = rand(tokens, D, seed=5), torch.zeros(H, D, device="cuda"), torch.zeros(H, device="cuda")
        stop = torch.cuda.synchronize if wait else (lambda: None)
        seen = []
        for _ in range(12):
            y, x8, rstd = norm.layer_norm_act8(x, g, b); stop()
            f, h8 = linear.linear_act(y, w1, b1, act="gelu_tanh", save="act8"); stop()
            linear.linear_act(f, w2, residual=x, out=x); stop()
            dh, a = linear.linear_act_dgrad(x, w2, h8, act="gelu_tanh", recompute=True); stop()
            linear.linear_bias_grad(dh, out=db, accumulate=True); stop()
            act8.act8_wgrad(dh, x8, weight=g, bias=b, dy_sum=db, out=dw, accumulate=True); stop()
            dy = linear.linear_act_dgrad(dh, w1, None); stop()
            dx, dg, dbeta = norm.layer_norm_act8_backward(dy, x8, g, rstd, residual_grad=x); stop()
            p8 = act8.act8_pack(dx); stop()
            x.copy_(act8.act8_unpack(p8) * 0.125); stop()
            seen += [dg, dbeta, act8.act8_unpack(p8)]
        return seen + [x, dw, db]

    for tokens in (1, 16, 130, T):
        one, other = chain(tokens, True), chain(tokens, False)
        assert all(torch.equal(p, q) for p, q in zip(one, other))
        assert all(torch.isfinite(p).all() for p in one)
    G.check_gemm_errors()


# few tiles on clusters with one and several chains, two waves of clusters, tiles cut into runs, unpacked and pairs
@pytest.mark.parametrize("T,N,K", [(512, 128, 128), (1000, 520, 328), (4100, 65, 200), (16384, 256, 256), (16384, 300, 2048), (16384, 512, 512),
                                   (2048, 1024, 1024), (300, 4096, 1024), (8192, 2048, 520)])
def test_act8_wgrad_either_way(T, N, K):
    """The way that is taken for these sizes, and a checkpoint that is converted tile by tile, with a gradient that is added to."""
    dy, x8, g, b, base = rand(T, N), act8.act8_pack(rand(T, K, seed=1)), rand(K, seed=2), rand(K, seed=3), rand(N, K, seed=4, dtype=F32)
    x, s = act8.act8_unpack(x8, F32).double(), linear.linear_bias_grad(dy)
    size = dy.double().abs().t() @ x.abs()
    want = base.double() + dy.double().t() @ (x * g.double() + b.double())
    slack = ((34 * 2.0 ** -23 + (T / 512 + 8) * 2.0 ** -24) * size * g.double().abs()
             + 2.0 ** -20 * dy.double().abs().sum(0)[:, None] * b.double().abs() + 2.0 ** -22 * (want.abs() + base.double().abs()))
    got = act8.act8_wgrad(dy, x8, weight=g, bias=b, dy_sum=s, out=base.clone(), accumulate=True)
    near(got, want, slack)
    for _ in range(3):
        assert torch.equal(got, act8.act8_wgrad(dy, x8, weight=g, bias=b, dy_sum=s, out=base.clone(), accumulate=True))
    if N % 8 == 0:
        out, stream = base.clone(), torch.cuda.current_stream().cuda_stream
        assert C.act8_wgrad(dy.data_ptr(), N, *x8.args(), out.data_ptr(), K, True, g.data_ptr(), b.data_ptr(), s.data_ptr(), T, N, K, 0,
                            G.workspace(0, stream).data_ptr(), G._err_flag(dy.device).data_ptr(), 2.0, stream) == 0
        near(out, want, slack)
    G.check_gemm_errors()


def test_products_of_two_streams_share_the_gpu():
    """Small and large products side by side: clusters of one stream, pairs of another, each as alone."""
    small = [(rand(t, 256, seed=t), rand(384, 256, seed=t + 1)) for t in (1, 16, 100)]
    large = [(rand(700, 512, seed=t), rand(2304, 512, seed=t + 1)) for t in (1, 2)]
    alone = [linear.linear_act(x, w, act="silu") for x, w in small + large]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    seen = [[], []]
    for _ in range(40):
        for s, cases, out in zip(streams, (small, large), seen):
            with torch.cuda.stream(s):
                out += [linear.linear_act(x, w, act="silu") for x, w in cases]
    torch.cuda.synchronize()
    for i, out in enumerate(seen[0]):
        assert torch.equal(out, alone[i % 3])
    for i, out in enumerate(seen[1]):
        assert torch.equal(out, alone[3 + i % 2])
    G.check_gemm_errors()


def test_rows_that_are_all_the_same_one():
    """Operands expanded from one row: every row at the same address."""
    one, w, dy = rand(1, 72), rand(40, 72, seed=1), rand(1, 40, seed=2)
    full = one.expand(5, 72)
    assert torch.equal(linear.linear_act(full, w), linear.linear_act(full.contiguous(), w))
    assert torch.equal(linear.linear_act(one, w[:1].expand(40, 72)), linear.linear_act(one, w[:1].expand(40, 72).contiguous()))
    assert torch.equal(linear.linear_act_dgrad(dy.expand(5, 40), w, None), linear.linear_act_dgrad(dy.expand(5, 40).contiguous(), w, None))
    x8 = act8.act8_pack(full)
    assert torch.equal(act8.act8_unpack(x8), act8.act8_unpack(act8.act8_pack(full.contiguous())))
    assert torch.equal(act8.act8_wgrad(dy.expand(5, 40), x8), act8.act8_wgrad(dy.expand(5, 40).contiguous(), x8))
    assert torch.equal(linear.linear_bias_grad(dy.expand(5, 40)), linear.linear_bias_grad(dy.expand(5, 40).contiguous()))
    got, want = (norm.layer_norm(v, one[0], one[0]) for v in (full, full.contiguous()))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    G.check_gemm_errors()


@pytest.mark.parametrize("M,N,K", [(4200, 1100, 136), (4200, 1098, 72), (4200, 1101, 72), (70, 44, 40), (70, 42, 40), (300, 41, 40)])
def test_linear_results_and_neighbours_on_any_boundary(M, N, K):
    """Residual, result, kept value and its gradient in matrices whose rows start on multiples of 8, 4 and 2 bytes: bit for bit what
    aligned ones give, and nothing written beside them."""
    x, w, b, res = rand(M, K), rand(N, K, seed=1), rand(N, seed=2), rand(M, N, seed=3)
    wide = lambda t: F.pad(t, (0, -N % 8))[:, :N]  # noqa: E731
    y, h = linear.linear_act(x, w, b, act="silu", residual=wide(res), save="bf16")
    assert y.stride(0) % 8 == 0 and h.stride(0) % 8 == 0
    room = torch.full((M * N + 16,), 7.0, dtype=BF, device="cuda")
    out = room[8:8 + M * N].view(M, N)
    assert torch.equal(linear.linear_act(x, w, b, act="silu", residual=res.contiguous(), out=out), y)
    assert (room[:8] == 7).all() and (room[8 + M * N:] == 7).all()
    cols = torch.full((M, N + 3), 7.0, dtype=BF, device="cuda")
    linear.linear_act(x, w, b, act="silu", residual=res, out=cols[:, 1:N + 1])
    assert torch.equal(cols[:, 1:N + 1], y) and (cols[:, 0] == 7).all() and (cols[:, N + 1:] == 7).all()
    near(linear.linear_act(x, w), x.double() @ w.double().t(), sum_slack(x.double(), w.double().t()))
    dy, w2 = rand(M, K, seed=4), rand(K, N, seed=5)
    one = linear.linear_act_dgrad(dy, w2, h, act="gelu", recompute=True)
    other = linear.linear_act_dgrad(dy, F.pad(w2, (0, -N % 8))[:, :N], h.contiguous(), act="gelu", recompute=True)
    assert all(torch.equal(p, q) for p, q in zip(one, other))
    G.check_gemm_errors()


@pytest.mark.parametrize("T,N,K", [(50, 2100, 1030), (50, 40, 203), (700, 2049, 1029), (20000, 257, 1035)])
def test_act8_wgrad_results_on_any_boundary(T, N, K):
    """Rows of the gradient that start on no 16-byte boundary, written and added to: bit for bit the aligned result."""
    dy, x8 = rand(T, N), act8.act8_pack(rand(T, K, seed=1))
    wide = torch.zeros(N, -(-K // 4) * 4, device="cuda")
    want = act8.act8_wgrad(dy, x8, out=wide[:, :K]).clone()
    room = torch.full((N * K + 8,), 7.0, device="cuda")
    got = act8.act8_wgrad(dy, x8, out=room[4:4 + N * K].view(N, K))
    assert torch.equal(got, want) and (room[:4] == 7).all() and (room[4 + N * K:] == 7).all()
    act8.act8_wgrad(dy, x8, out=wide[:, :K], accumulate=True)
    assert torch.equal(act8.act8_wgrad(dy, x8, out=got, accumulate=True), wide[:, :K])
    G.check_gemm_errors()


@pytest.mark.parametrize("rows,d", [(5, 2), (700, 34), (3000, 534), (700, 2050), (3, 4102), (2, 8190), (3000, 1003)])
def test_layer_norm_rows_on_few_bytes(rows, d):
    """Rows that start on multiples of 4 or 2 bytes, in pairs and one by one, with and without 8-bit rows; and the same rows inside
    wider ones, at an offset: the result does not depend on where they lie, nothing beside it is read into it."""
    test_layer_norm_forward(rows, d, BF)
    for join in (False, True):
        test_layer_norm_backward(rows, d, join, BF)
    x, dy, g = rand(rows, d) * 3 + 1, rand(rows, d, seed=3), rand(d, seed=1)
    y, mean, rstd = norm.layer_norm(x, g)
    want = norm64_grads(dy, norm64(x, g, torch.zeros_like(g))[3], rstd.double(), g, None)
    for start, room in ((1, 3), (2, 4)):
        def inside(t):
            w = torch.full((rows, d + room), math.nan, dtype=BF, device="cuda")
            w[:, start:start + d] = t
            return w[:, start:start + d]
        xs, dys = inside(x), inside(dy)
        ys, means, rstds = norm.layer_norm(xs, g)
        # sums in another order: a value that lies on the edge of two bf16 may go the other way
        assert ((ys.double() - y.double()).abs() <= 2.0 ** -7 * y.double().abs() + 2.0 ** -18).all() and torch.isfinite(means).all()
        y8, x8, r8 = norm.layer_norm_act8(xs, g)
        assert torch.equal(y8, ys) and torch.equal(r8, rstds)
        for dx, dw, db in (norm.layer_norm_backward(dys, xs, g, means, rstds), norm.layer_norm_act8_backward(dys, x8, g, r8)):
            assert all(torch.isfinite(t).all() for t in (dx, dw, db))
            near(db, want[2], 2.0 ** -20 * dy.double().abs().sum(0))
