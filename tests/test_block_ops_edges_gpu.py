"""Block operators where values, sizes or settings reach an edge: the largest steps of the 8-bit format on every way that the weight
gradient takes, a limit on the CTAs of products, rows anywhere in memory. Against 64 bits, with the bounds of ``test_block_ops_gpu``."""
import pytest
import torch

from parameter_server_b200._lib import C
from parameter_server_b200.ops import act8, linear, norm
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


# ---- a limit on the CTAs of products ----------------------------------------------------------------------------------------

def ctas_of(call):
    """Of the products' kernels that `call` launches (the memory passes have fewer threads): CTAs, and how many there are."""
    from cuda.bindings import driver

    def ok(result):
        assert result[0] == driver.CUresult.CUDA_SUCCESS, result[0]
        return result[1:] if len(result) > 2 else result[-1]

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw = driver.CUgraph(graph.raw_cuda_graph())
    count = ok(driver.cuGraphGetNodes(raw))[-1]
    nodes = ok(driver.cuGraphGetNodes(raw, count))[0][:count]
    kernels = [ok(driver.cuGraphKernelNodeGetParams(n)) for n in nodes
               if ok(driver.cuGraphNodeGetType(n)) == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL]
    return [k.gridDimX * k.gridDimY * k.gridDimZ for k in kernels if k.blockDimX >= 384]


def sum_bound(a, b):
    """a [M, K], b [K, N] in 64 bits: the tensor core cuts its sum off once per 16 products."""
    return (a.shape[1] / 16 + 2) * 2.0 ** -23 * (a.abs() @ b.abs())


@pytest.mark.parametrize("limit", [2, 17, 32, 100])
# few tokens, more of them, many; input gradients; weight gradients on clusters, unpacked, and converted
@pytest.mark.parametrize("kind,M,N,K", [("forward", 1, 300, 200), ("forward", 16, 8192, 512), ("forward", 128, 2048, 2048), ("forward", 512, 2048, 2048),
                                        ("forward", 1024, 4096, 1024), ("dgrad", 64, 8192, 1024), ("dgrad", 700, 1000, 520), ("wgrad", 4096, 512, 512),
                                        ("wgrad", 1000, 4096, 1024), ("wgrad", 4096, 1536, 2048)])
def test_products_keep_to_the_limit_of_ctas(kind, M, N, K, limit):
    if kind == "wgrad":
        dy, x8 = rand(M, N), act8.act8_pack(rand(M, K, seed=1))
        a, b = dy.double().t(), act8.act8_unpack(x8, F32).double()
        call, slack = (lambda: act8.act8_wgrad(dy, x8)), (34 * 2.0 ** -23 + (M / 512 + 8) * 2.0 ** -24) * (a.abs() @ b.abs())
    else:
        x, w = rand(M, K), rand(N, K, seed=1, std=K ** -0.5)
        a, b = x.double(), w.double().t()
        call, slack = (lambda: linear.linear_act(x, w)), sum_bound(a, b)
        if kind == "dgrad":
            wt = w.t().contiguous()
            call = lambda: linear.linear_act_dgrad(x, wt, None)  # noqa: E731
    C.gemm_set_cta_limit(limit)
    try:
        got = call()
        grids = ctas_of(call)
    finally:
        C.gemm_set_cta_limit(0)
    assert len(grids) == 1 and grids[0] <= limit, grids
    want = a @ b
    assert ((got.double() - want).abs() <= slack + (2.0 ** -8 if got.dtype == BF else 2.0 ** -23) * want.abs()).all()
    free = call()   # without a limit: the same sums, perhaps in another order
    assert ((free.double() - want).abs() <= slack + (2.0 ** -8 if got.dtype == BF else 2.0 ** -23) * want.abs()).all()
    G.check_gemm_errors()


# ---- a result in the residual's place ---------------------------------------------------------------------------------------

# pairs and clusters; rows that share 32-byte sectors, lines, or neither with their neighbours' tiles
@pytest.mark.parametrize("M,N,K,start", [(2048, 2048, 512, 0), (2048, 2040, 512, 8), (700, 1000, 512, 8), (16, 2048, 512, 0), (300, 520, 256, 4)])
def test_a_result_in_the_residuals_place_call_after_call(M, N, K, start):
    """Each launch reads what the one before wrote, over the same memory, and begins beside its tail: as if it were done one by one."""
    x, ws = rand(M, K), [rand(N, K, seed=s, std=K ** -0.5) for s in range(1, 4)]

    def chain(wait):
        room = torch.zeros(M, N + 24, dtype=BF, device="cuda")
        res = room[:, start:start + N]
        for k in range(12):
            linear.linear_act(x, ws[k % 3], act="silu", residual=res, out=res)
            if wait:
                torch.cuda.synchronize()
        assert (room[:, :start] == 0).all() and (room[:, start + N:] == 0).all()
        return res.clone()

    want = chain(True)
    for _ in range(3):
        assert torch.equal(chain(False), want)
    G.check_gemm_errors()


# ---- layer norm on rows inside wider ones -----------------------------------------------------------------------------------

def inside(t, start, room):
    """The same rows at a column `start` of rows `room` wider, among NaN."""
    rows, d = t.shape
    wide = torch.full((rows, d + room), float("nan"), dtype=t.dtype, device="cuda")
    wide[:, start:start + d] = t
    return wide[:, start:start + d]


def within(got, want, slack):
    one = 2.0 ** -8 if got.dtype == BF else 2.0 ** -23
    off = (got.double() - want).abs()
    assert (off <= one * want.abs() + slack + 1e-30).all(), (off / (one * want.abs() + slack + 1e-30)).max()


# start 1 of 3 more: rows on every 2-byte boundary; 2 of 4: on 4 bytes; 8 of 8: on 16; and mixed, so that operands differ
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("places", [(1, 3), (2, 4), (8, 8), "mixed"])
@pytest.mark.parametrize("rows,d", [(5, 2), (700, 34), (3000, 534), (700, 1001), (700, 2050), (3, 4102), (2, 8190), (640, 2048), (2, 8200)])
def test_layer_norm_of_rows_inside_wider_ones(rows, d, places, dtype):
    """Forward and backward, from x and from 8-bit rows, with a residual gradient: each value against 64 bits."""
    at = [(1, 3), (2, 4), (0, 2), (3, 5)] if places == "mixed" else [places] * 4
    x, dy, join = rand(rows, d, dtype=dtype) * 3 + 1, rand(rows, d, seed=3, dtype=dtype), rand(rows, d, seed=4, dtype=dtype)
    g, b = rand(d, seed=1, dtype=dtype), rand(d, seed=2, dtype=dtype)
    xs, dys, js = inside(x, *at[0]), inside(dy, *at[1]), inside(join, *at[2])
    gs = inside(g.view(1, d), *at[3])[0]
    y, mean, rstd = norm.layer_norm(xs, gs, b)
    x64 = x.double()
    dev = (x64.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt()
    xhat = (x64 - x64.mean(1, keepdim=True)) / dev
    # x and the mean enter with 2^-24 of the largest |x| over the deviation, the sums' roundings stay below 2^-20 of the values
    off = 2.0 ** -22 * x64.abs().amax(1, keepdim=True) / dev + 2.0 ** -20 * (1 + xhat.abs())
    within(y, xhat * g.double() + b.double(), off * (1 + g.double().abs()))
    y8, x8, rstd8 = norm.layer_norm_act8(xs, gs, b)
    assert torch.equal(y8, y) and torch.equal(rstd8, rstd)
    stats = (x64 - mean.double()[:, None]) * rstd.double()[:, None]
    p = dy.double() * g.double()
    for hat, result in ((stats, norm.layer_norm_backward(dys, xs, gs, mean, rstd, residual_grad=js)),
                        (act8.act8_unpack(x8, F32).double(), norm.layer_norm_act8_backward(dys, x8, gs, rstd, residual_grad=js))):
        dx, dw, db = result
        want = rstd.double()[:, None] * (p - p.mean(1, keepdim=True) - hat * (p * hat).mean(1, keepdim=True)) + join.double()
        size = p.abs() + p.abs().mean(1, keepdim=True) + hat.abs() * (p * hat).abs().mean(1, keepdim=True)
        within(dx, want, 2.0 ** -20 * rstd.double()[:, None] * size + 2.0 ** -24 * want.abs())
        within(dw, (dy.double() * hat).sum(0), 2.0 ** -20 * (dy.double() * hat).abs().sum(0))
        within(db, dy.double().sum(0), 2.0 ** -20 * dy.double().abs().sum(0))
