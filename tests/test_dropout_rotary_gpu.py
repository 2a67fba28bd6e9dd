"""Dropout and rotary positions against plain implementations in 64 bits, value by value.

Bounds. Dropout: the mask is equal; a kept value is off by the rounding of its factor and of the product in fp32 (2^-23 of it together), the
sum and the result by one rounding each. Rotary: the fraction of a turn is rounded to fp32 (2^-26 turns, 2^-23.3 radians), CUDA's sincospif is
off by 2 units of 2^-24 at most, a product's factor, the two products and the sum are rounded (2^-24 of |x| + |y| each): 2^-21 together; the
angle's product in 64 bits has three roundings on each side, 2^-50 of the angle together."""
import math

import philox64
import pytest
import torch

from parameter_server_b200.ops import dropout, rotary

pytestmark = pytest.mark.gpu

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HALF_STEP = {BF: 2.0 ** -8, F32: 2.0 ** -24}


def rand(*shape, seed=0, std=1.0, dtype=BF):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * len(shape) + sum(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def near(got, want, slack):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    bound = HALF_STEP[got.dtype] * want.abs() + slack + 1e-37
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the bound"


# ---- dropout -----------------------------------------------------------------------------------------------------------

def dropped(x, p, seed, offset):
    rows, cols = x.shape
    mask = torch.from_numpy(philox64.kept(rows, cols, p, seed, offset)).cuda()
    return torch.where(mask, x.double() * philox64.grown(p), torch.zeros_like(x, dtype=F64)), mask


def check_dropout(x, p, seed, offset, residual=None, out=None):
    x2 = x.reshape(-1, x.shape[-1]).clone()
    want, mask = dropped(x2, p, seed, offset)
    slack = 2.0 ** -23 * want.abs()
    if residual is not None:
        want = want + residual.reshape(want.shape).double()
        slack = slack + 2.0 ** -24 * want.abs()
    got = dropout.dropout(x, p, seed, offset, residual=residual, out=out)
    assert got.dtype == x.dtype and got.shape == x.shape
    near(got.reshape(want.shape), want, slack)
    return got, mask


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 3), (3, 4), (5, 7), (2, 8), (17, 33), (4, 2048), (1000, 96), (129, 1001), (3, 20000), (40001, 4)])
@pytest.mark.parametrize("residual", [False, True])
def test_dropout_is_its_mask(rows, cols, residual, dtype):
    x, r = rand(rows, cols, dtype=dtype), rand(rows, cols, seed=1, dtype=dtype) if residual else None
    got, mask = check_dropout(x, 0.3, 0x123456789ABCDEF0, 5, r)
    if r is None:
        assert (got[~mask] == 0).all()
    near(dropout.dropout_backward(x, 0.3, 0x123456789ABCDEF0, 5), dropped(x, 0.3, 0x123456789ABCDEF0, 5)[0], 2.0 ** -23 * x.double().abs() * 2)


@pytest.mark.parametrize("rows,cols", [(2500, 2048), (2500, 2056), (5001, 1001), (4001, 1302), (3001, 1636), (700001, 8), (620001, 9), (1300001, 5), (5000001, 1), (1, 5000003)])
def test_dropout_of_many_values(rows, cols):
    """32 bytes of a thread at a time, on every boundary, with every end of a row."""
    x, r = rand(rows, cols), rand(rows, cols, seed=1)
    check_dropout(x, 0.3, 77, 6, r)
    wide = torch.full((rows, cols + 3), 7.0, dtype=BF, device="cuda")
    got, mask = check_dropout(x, 0.3, 77, 6, out=wide[:, 1:cols + 1])
    assert (got[~mask] == 0).all() and (wide[:, 0] == 7).all() and (wide[:, cols + 1:] == 7).all()
    want = got.clone()
    assert torch.equal(dropout.dropout(x, 0.3, 77, 6, out=x), want)   # in place


@pytest.mark.parametrize("p", [0.0, 2.0 ** -32, 1e-3, 0.5, 0.9, 1 - 2.0 ** -20])
def test_every_share(p):
    x = rand(64, 257) + 4
    got, mask = check_dropout(x, p, 99, 1 << 40)
    if p == 0:
        assert torch.equal(got, x)
    n = x.numel()
    assert abs(mask.sum().item() - n * (1 - p)) <= 6 * math.sqrt(n * p * (1 - p)) + 1


@pytest.mark.parametrize("seed,offset", [(0, 0), (-1, 0), ((1 << 64) - 1, (1 << 64) - 1), (1 << 32, 1 << 32), (7, 8)])
def test_seeds_and_offsets(seed, offset):
    check_dropout(rand(9, 130), 0.4, seed, offset)


def test_a_seed_in_memory_is_read_when_the_kernel_runs():
    x = rand(33, 100)
    seed = torch.tensor([-5], device="cuda")
    assert torch.equal(dropout.dropout(x, 0.3, seed, 3), dropout.dropout(x, 0.3, -5, 3))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        dropout.dropout(x, 0.3, seed, 3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        seed.add_(1)
        y = dropout.dropout(x, 0.3, seed, 3)
    for k in (1, 2):
        graph.replay()
        assert torch.equal(y, dropout.dropout(x, 0.3, -5 + k, 3))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_in_memory_in_any_way(dtype):
    base, r = rand(60, 300, dtype=dtype), rand(60, 300, seed=2, dtype=dtype)
    for cut in ((slice(None), slice(0, 256)), (slice(None), slice(1, 200)), (slice(0, 60, 3), slice(2, 131)), (slice(None), slice(4, 260)), (slice(5, 6), slice(8, 264))):
        x, res = base[cut], r[cut]
        assert torch.equal(dropout.dropout(x, 0.2, 11, 1, residual=res), dropout.dropout(x.contiguous(), 0.2, 11, 1, residual=res.contiguous()))
        check_dropout(x, 0.2, 11, 1, res)
        wide = torch.full((60, 300), 7.0, dtype=dtype, device="cuda")
        out = wide[cut]
        dropout.dropout(x, 0.2, 11, 1, residual=res, out=out)
        assert torch.equal(out, dropout.dropout(x, 0.2, 11, 1, residual=res))
        out.fill_(7.0)
        assert (wide == 7).all()   # nothing beside the rows was written
    three = rand(4, 5, 64, dtype=dtype)
    assert torch.equal(dropout.dropout(three, 0.2, 11), dropout.dropout(three.view(20, 64), 0.2, 11).view(4, 5, 64))
    across = rand(64, 32, dtype=dtype).t()
    assert torch.equal(dropout.dropout(across, 0.2, 11), dropout.dropout(across.contiguous(), 0.2, 11))
    assert torch.equal(dropout.dropout(x[:1].expand(9, -1), 0.2, 11), dropout.dropout(x[:1].expand(9, -1).contiguous(), 0.2, 11))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("cols", [256, 101])
def test_results_in_the_inputs_place(cols, dtype):
    x, r = rand(77, cols, dtype=dtype), rand(77, cols, seed=3, dtype=dtype)
    want = dropout.dropout(x, 0.3, 1, residual=r)
    into, over = r.clone(), x.clone()
    assert dropout.dropout(x, 0.3, 1, residual=into, out=into) is into and torch.equal(into, want)
    assert dropout.dropout(over, 0.3, 1, residual=r, out=over) is over and torch.equal(over, want)


def test_what_is_dropped_counts_as_nothing():
    x = rand(50, 200)
    mask = torch.from_numpy(philox64.kept(50, 200, 0.5, 4, 0)).cuda()
    x[~mask] = math.nan
    x[0][~mask[0]] = math.inf
    got = dropout.dropout(x, 0.5, 4)
    assert torch.isfinite(got).all() and (got[~mask] == 0).all()
    y = rand(50, 200)
    y[mask] = math.nan
    assert torch.equal(torch.isnan(dropout.dropout(y, 0.5, 4)), mask)


def test_dropout_of_nothing():
    for shape in ((0, 8), (4, 0), (0,), (2, 0, 8)):
        assert dropout.dropout(torch.empty(shape, dtype=BF, device="cuda"), 0.5, 1).shape == shape


def test_dropout_differs_between_rows_columns_and_offsets():
    x = torch.ones(256, 256, device="cuda")
    a = dropout.dropout(x, 0.5, 1, 0) != 0
    assert 0.45 < (a[1:] ^ a[:-1]).float().mean() < 0.55 and 0.45 < (a[:, 1:] ^ a[:, :-1]).float().mean() < 0.55
    assert 0.45 < (a ^ (dropout.dropout(x, 0.5, 1, 1) != 0)).float().mean() < 0.55
    assert 0.45 < (a ^ (dropout.dropout(x, 0.5, 2, 0) != 0)).float().mean() < 0.55


def test_more_values_than_32_bits_count():
    """Rows behind element 2^32 (fp32: behind byte 2^34) are read, drawn and written in their own place."""
    rows, cols = 65600, 65536
    x = torch.ones(rows, cols, dtype=BF, device="cuda")
    y = dropout.dropout(x, 0.5, 21, out=x)
    for row in (0, 32768, 65535, 65536, rows - 1):
        mask = torch.from_numpy(philox64.kept(1, cols, 0.5, 21, 0, first_row=row)).cuda()
        assert torch.equal(y[row:row + 1], mask.to(BF) * 2)


# ---- rotary positions --------------------------------------------------------------------------------------------------

def turned(x, freqs, pos, interleaved, scale, back=False):
    """(result, |x| + |y| of each value's pair) for [batch, tokens, heads, dim], positions [batch, tokens]."""
    angle = pos.double().unsqueeze(-1) * freqs
    c, s = (scale * angle.cos()).unsqueeze(2), (scale * angle.sin()).unsqueeze(2) * (-1 if back else 1)
    n = freqs.numel()
    out, size = x.double().clone(), torch.zeros_like(x, dtype=F64)
    lo, hi = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., lo].double(), x[..., hi].double()
    out[..., lo], out[..., hi] = a * c - b * s, a * s + b * c
    slack = scale * (a.abs() + b.abs()) * (2.0 ** -21 + 2.0 ** -50 * angle.abs().unsqueeze(2))
    size[..., lo] = size[..., hi] = slack
    return out, size


def check_rotary(q, k, freqs, pos=None, interleaved=False, scale=1.0, offset=0, **out):
    """Forward and backward."""
    four = lambda x: x if x.dim() == 4 else x.unsqueeze(0)  # noqa: E731
    B, T = four(q).shape[:2]
    at = (torch.arange(T, device="cuda") if pos is None else pos.long()) + offset
    at = at.expand(B, T) if at.dim() == 1 or at.shape[0] == 1 else at
    if out:
        q, k = q.clone(), k.clone()
    for call, back in ((rotary.rotary, False), (rotary.rotary_backward, True)):
        got = call(q, k, freqs, pos, offset=offset, interleaved=interleaved, scale=scale, **out)
        for x, y in zip((q,) if k is None else (q, k), (got,) if k is None else got):
            want, slack = turned(four(x), freqs, at, interleaved, scale, back)
            assert y.shape == x.shape and y.dtype == x.dtype
            near(four(y), want, slack)
            assert torch.equal(y[..., 2 * freqs.numel():], x[..., 2 * freqs.numel():])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(2, 2), (8, 8), (16, 6), (64, 64), (80, 80), (76, 50), (128, 128), (128, 32), (96, 96), (33, 14), (256, 256), (7, 0), (700, 600)])
def test_rotary(dim, rot, interleaved, dtype):
    freqs = rotary.rotary_frequencies(rot)[0] if rot else torch.empty(0, dtype=F64, device="cuda")
    check_rotary(rand(3, 37, 5, dim, dtype=dtype), rand(3, 37, 2, dim, seed=1, dtype=dtype), freqs, interleaved=interleaved)


@pytest.mark.parametrize("batch,tokens,hq,hk", [(1, 1, 1, 1), (1, 1, 32, 8), (64, 1, 16, 16), (1, 3000, 1, 0), (2, 257, 40, 8), (7, 5, 3, 1), (1, 1, 300, 2)])
def test_heads_and_tokens(batch, tokens, hq, hk):
    freqs = rotary.rotary_frequencies(64)[0]
    k = rand(batch, tokens, hk, 64, seed=1) if hk else None
    check_rotary(rand(batch, tokens, hq, 64), k, freqs, offset=13)
    check_rotary(rand(tokens, hq, 64), None if k is None else k[0], freqs)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_positions(dtype):
    q, k = rand(3, 20, 4, 32, dtype=dtype), rand(3, 20, 2, 32, seed=1, dtype=dtype)
    freqs = rotary.rotary_frequencies(32)[0]
    g = torch.Generator(device="cuda").manual_seed(3)
    far = torch.randint(-(1 << 31), 1 << 31, (3, 20), generator=g, device="cuda")
    far[0, 0], far[0, 1], far[1, 0] = (1 << 31) - 1, -(1 << 31), 0
    for pos in (far, far.int(), far[:1], far[0], far[0].int(), far.t().contiguous().t(), far[0, :1].expand(20)):
        check_rotary(q, k, freqs, pos)
    check_rotary(q, k, freqs, far, offset=1 << 33)
    check_rotary(q, k, freqs, offset=-100)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(8, 2), (8, 6), (40, 38), (64, 2), (96, 50), (192, 130), (256, 254), (1024, 1022), (2048, 6), (4096, 10)])
@pytest.mark.parametrize("batch,tokens,hq,hk", [(1, 1, 1, 0), (2, 130, 5, 2), (1, 700, 40, 8)])
def test_parts_of_heads_on_whole_blocks(batch, tokens, hq, hk, dim, rot, interleaved, dtype):
    """Heads of whole 16-byte blocks whose halves, or whose turning part, end inside one; also in place."""
    freqs = rotary.rotary_frequencies(rot)[0]
    qkv = rand(batch, tokens, hq + hk + 1, dim, dtype=dtype)
    q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hk] if hk else None
    check_rotary(q, k, freqs, interleaved=interleaved, offset=3, scale=1.5)
    want = rotary.rotary(q, k, freqs, interleaved=interleaved)
    last = qkv[:, :, -1].clone()
    rotary.rotary(q, k, freqs, interleaved=interleaved, out_q=q, out_k=k)
    assert torch.equal(q, want[0] if hk else want) and (not hk or torch.equal(k, want[1])) and torch.equal(qkv[:, :, -1], last)


def test_values_that_do_not_turn_keep_their_bits():
    x = torch.zeros(1, 3, 2, 16, dtype=BF, device="cuda")
    x.view(torch.int16)[..., 6:] = torch.tensor([0x7FC1, -1, 0x7F80, -0x80, 0x0001, -0x8000, 0x7FFF, 5, 6, 7], dtype=torch.int16, device="cuda")
    for interleaved in (False, True):
        y = rotary.rotary(x, None, rotary.rotary_frequencies(6)[0], interleaved=interleaved)
        assert torch.equal(y.view(torch.int16)[..., 6:], x.view(torch.int16)[..., 6:])


def test_scaled_frequencies():
    q, k = rand(1, 50, 4, 128), rand(1, 50, 4, 128, seed=1)
    for scaling in ("linear", "ntk", "yarn"):
        freqs, scale = rotary.rotary_frequencies(128, scaling=scaling, factor=8.0, trained_length=4096)
        check_rotary(q, k, freqs, scale=scale, offset=30000)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(64, 64), (64, 24), (20, 20), (36, 22)])
def test_heads_in_memory_in_any_way(dim, rot, interleaved, dtype):
    freqs = rotary.rotary_frequencies(rot)[0]
    qkv = rand(2, 19, 9, dim, dtype=dtype)
    ways = [
        (qkv[:, :, :4], qkv[:, :, 4:6]),                                                                          # a packed product
        (rand(2, 4, 19, dim, dtype=dtype).transpose(1, 2), rand(2, 2, 19, dim, dtype=dtype).transpose(1, 2)),     # heads ahead of tokens
        (qkv[:, ::2, ::3], qkv[:, 1::2, 1::4][:, :9].repeat(1, 2, 1, 1)[:, :10]),                                  # steps
        (rand(2, 19, 4, dim + 3, dtype=dtype)[..., 1:dim + 1], rand(2, 19, 2, dim + 8, dtype=dtype)[..., 8:]),     # rows on other boundaries
        (rand(2, 19, 1, dim, dtype=dtype).expand(-1, -1, 4, -1), rand(1, 1, 2, dim, dtype=dtype).expand(2, 19, -1, -1)),
        (rand(2, 19, dim, 4, dtype=dtype).transpose(2, 3), rand(2, 19, dim, 2, dtype=dtype).transpose(2, 3)),     # copied
    ]
    for q, k in ways:
        check_rotary(q, k, freqs, interleaved=interleaved, offset=9)
        room = torch.full((2, q.shape[1], 9, dim + 5), 7.0, dtype=dtype, device="cuda")
        oq, ok = room[:, :, 1:1 + q.shape[2], 2:2 + dim], room[:, :, 6:6 + k.shape[2], 2:2 + dim]
        check_rotary(q, k, freqs, interleaved=interleaved, out_q=oq, out_k=ok)
        oq.fill_(7.0)
        ok.fill_(7.0)
        assert (room == 7).all()   # nothing beside the heads was written


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(64, 64), (64, 24), (33, 14)])
def test_rotary_in_place(dim, rot, interleaved, dtype):
    freqs = rotary.rotary_frequencies(rot)[0]
    qkv = rand(2, 50, 12, dim, dtype=dtype)
    want, before = qkv.clone(), qkv.clone()
    want[:, :, :8], want[:, :, 8:10] = rotary.rotary(qkv[:, :, :8], qkv[:, :, 8:10], freqs, interleaved=interleaved)
    q, k = qkv[:, :, :8], qkv[:, :, 8:10]
    rotary.rotary(q, k, freqs, interleaved=interleaved, out_q=q, out_k=k)
    assert torch.equal(qkv, want) and torch.equal(qkv[:, :, 10:], before[:, :, 10:])


def test_values_that_are_not_finite_stay_in_their_pairs():
    q = torch.ones(1, 4, 2, 8, device="cuda")
    q[0, 1, 0, 2] = math.nan
    q[0, 2, 1, 5] = math.inf
    got = rotary.rotary(q, None, rotary.rotary_frequencies(8)[0])
    bad = ~torch.isfinite(got)
    assert bad[0, 1, 0].nonzero().flatten().tolist() == [2, 6] and bad[0, 2, 1].nonzero().flatten().tolist() == [1, 5] and bad.sum() == 4


def test_turning_back():
    """The gradient is the transpose: <R x, y> = <x, R' y>; forward and back again multiplies by scale^2."""
    q, y = rand(2, 30, 4, 64, dtype=F32), rand(2, 30, 4, 64, seed=1, dtype=F32)
    freqs = rotary.rotary_frequencies(48)[0]
    fwd, bwd = rotary.rotary(q, None, freqs, scale=1.25), rotary.rotary_backward(y, None, freqs, scale=1.25)
    assert abs((fwd.double() * y).sum() - (q.double() * bwd).sum()) <= 2.0 ** -20 * (fwd.double() * y).abs().sum()
    there = rotary.rotary_backward(fwd, None, freqs, scale=1 / 1.25)
    # (two passes: 2 * 2^-21 of |x| + |y|, each below 5)
    assert ((there - q).abs() <= 2.0 ** -20 * 10).all()


def test_rotary_of_nothing():
    f = rotary.rotary_frequencies(8)[0]
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8), (0, 2, 8)):
        x = torch.empty(shape, dtype=BF, device="cuda")
        assert rotary.rotary(x, x, f)[0].shape == shape


def test_far_into_a_long_cache():
    """Offsets behind element 2^32."""
    tokens, heads, dim = 270000, 128, 128
    x = torch.zeros(tokens, heads, dim, dtype=BF, device="cuda")
    rows = [0, 131071, 262143, 262144, tokens - 1]
    some = rand(len(rows), heads, dim)
    x[rows] = some
    freqs = rotary.rotary_frequencies(dim)[0]
    rotary.rotary(x, None, freqs, out_q=x)
    want, slack = turned(some.unsqueeze(0), freqs, torch.tensor([rows], device="cuda"), False, 1.0)
    near(x[rows].unsqueeze(0), want, slack)


def test_both_under_a_graph_and_on_another_stream():
    x, q = rand(300, 512), rand(1, 300, 4, 64)
    freqs = rotary.rotary_frequencies(64)[0]
    want = dropout.dropout(x, 0.1, 3), rotary.rotary(q, None, freqs)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = dropout.dropout(x, 0.1, 3), rotary.rotary(q, None, freqs)
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = dropout.dropout(x, 0.1, 3), rotary.rotary(q, None, freqs)
    x.mul_(2)
    q.mul_(2)
    graph.replay()
    assert all(torch.equal(a, 2 * b) for a, b in zip(got, want))
