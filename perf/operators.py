"""The operators of a decoder block in training, as timed cases: layer norm, the linear layer with its epilogue, and
activation checkpoints in 8 bits with the backward passes that read them.

A case is a dict of plain values; ``prepare`` makes what a program holds before the call, ``run`` is one pass: the plain
form (elementary torch operations in 32 bits, rounded once at the end), or, where ``own`` is set, the calls into the
package. ``exact`` is the same in 64 bits, ``work`` what a pass cannot do without.

Kinds:

* ``norm``      layer norm forward (``bwd`` false: y, mean, rstd) or backward (``bwd`` true: dx, dweight, dbias); ``join``
  adds the gradient that the residual branch brings to dx. ``pad``: extra columns between the rows of x in memory.
* ``norm8``     a layer norm whose normalised rows are kept in 8 bits between the passes: forward (y, the checkpoint as the
  values it stands for, rstd), or backward from a checkpoint.
* ``linear``    act(x w^T + b) + residual, with the value before the activation in bf16 too where ``save`` asks for it.
* ``mlp``       the hidden layer of a transformer's MLP in training: act(x w1^T + b1) with a checkpoint of the value before the
  activation in ``bits`` bits, then the backward pass into it, (dy w2) * act'(h), with act(h) formed again from the checkpoint.
* ``wgrad8``    dw = dy^T x with x a checkpoint in 8 bits. ``pack``: the pass makes the checkpoint first. ``norm``: x is a layer
  norm's output, rebuilt from its normalised rows in 8 bits (x8 * gamma + beta). ``acc``: added to a gradient that is there.

An 8-bit checkpoint holds 32 neighbours of a row as whole numbers of -127..127 and one power of two: the smallest step
2^(e-127), e in 1..249, at which the largest of them rounds to at most 127; e = 255 marks a block that held an infinity or NaN.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5
BLOCK = 32


def listed():
    return [
        # scoring a handful of tokens: one norm between two small products, where the launch is most of the time
        dict(name="norm_fwd_16", kind="norm", bwd=False, rows=16, d=2048, dtype="bf16", pad=0, join=False),
        # backward on one training micro-batch of the decoder (8 sequences of 2048 tokens, d_model 2048), where the gradient of
        # the residual branch joins
        dict(name="norm_bwd_16k", kind="norm", bwd=True, rows=16384, d=2048, dtype="bf16", pad=0, join=True),
        # a model kept in 32 bits with an odd width and rows that are not packed
        dict(name="norm_bwd_odd_f32", kind="norm", bwd=True, rows=4099, d=1001, dtype="f32", pad=3, join=False),
        # the same micro-batch with its normalised rows kept in 8 bits, forward
        dict(name="norm8_fwd_16k", kind="norm8", bwd=False, rows=16384, d=2048, pad=0, join=False),
        # and backward from them
        dict(name="norm8_bwd_16k", kind="norm8", bwd=True, rows=16384, d=2048, pad=0, join=True),
        # the first layer of the MLP for 16 tokens: as fast as its weights are read
        dict(name="linear_16", kind="linear", tokens=16, n=8192, k=2048, act="gelu_tanh", bias=True, res=False, save=False),
        # odd sizes, another activation, a residual and the value before the activation kept
        dict(name="linear_odd", kind="linear", tokens=1025, n=1000, k=776, act="gelu", bias=True, res=True, save=True),
        # the second layer of the decoder's MLP on a micro-batch, back into the residual stream
        dict(name="linear_out_16k", kind="linear", tokens=16384, n=2048, k=8192, act="none", bias=True, res=True, save=False),
        # the hidden layer for half a sequence, forward and backward, checkpoint in bf16
        dict(name="mlp_1k", kind="mlp", tokens=1024, n=8192, k=2048, act="gelu_tanh", bits=16),
        # the hidden layer on a micro-batch with its checkpoint in 8 bits
        dict(name="mlp8_16k", kind="mlp", tokens=16384, n=8192, k=2048, act="gelu_tanh", bits=8),
        # the weight gradient of the QKV layer from the norm's 8-bit checkpoint
        dict(name="wgrad8_qkv_16k", kind="wgrad8", tokens=16384, n=6144, k=2048, pack=False, norm=True, acc=False),
        # odd sizes, checkpoint made in the same pass, second micro-batch of an accumulation
        dict(name="wgrad8_odd", kind="wgrad8", tokens=1000, n=520, k=328, pack=True, norm=False, acc=True),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    kind = rng.choice(["norm", "norm8", "linear", "linear", "mlp", "wgrad8", "wgrad8"])
    if kind in ("norm", "norm8"):
        d = log(64, 8192)
        if rng.random() < 0.5:
            d = max(64, d // 64 * 64)
        rows = log(1, max(1, min(40000, 16384 * 2048 // d)))
        bwd = rng.random() < 0.5
        if kind == "norm8":
            return dict(kind=kind, bwd=bwd, rows=rows, d=d, pad=rng.choice([0, 0, 8, 40]), join=bwd and rng.random() < 0.5)
        return dict(kind=kind, bwd=bwd, rows=rows, d=d, dtype=rng.choice(["bf16", "bf16", "f32"]), pad=rng.choice([0, 0, 5, 8]), join=bwd and rng.random() < 0.5)
    n, k = log(128, 8192), log(128, 8192)
    if rng.random() < 0.7:
        n, k = -(-n // 8) * 8, -(-k // 8) * 8
    most = 16384 * 8192 * 2048 // (n * k)
    tokens = log(1, max(1, min(16384, most)))
    if kind == "linear":
        return dict(kind=kind, tokens=tokens, n=n, k=k, act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), bias=rng.random() < 0.7, res=rng.random() < 0.5, save=rng.random() < 0.4)
    if kind == "mlp":
        return dict(kind=kind, tokens=tokens, n=n, k=k, act=rng.choice(["relu", "gelu", "gelu_tanh", "silu"]), bits=rng.choice([8, 8, 16]))
    norm = rng.random() < 0.4
    return dict(kind=kind, tokens=tokens, n=n, k=k, pack=not norm and rng.random() < 0.6, norm=norm, acc=rng.random() < 0.4)


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _stream_rows(gen, rows, d, pad, dtype):
    """Rows as a residual stream has them: channels of different size, a few of them large, not centred."""
    scale = torch.exp(0.5 * torch.randn(d, generator=gen, device="cuda"))
    scale[torch.randint(0, d, (max(1, d // 256),), generator=gen, device="cuda")] *= 12
    x = torch.empty(rows, d + pad, dtype=dtype, device="cuda")
    x.copy_(torch.randn(rows, d + pad, generator=gen, device="cuda"))
    x = x[:, :d]
    x.mul_(scale.to(dtype)).add_((0.3 * torch.randn(d, generator=gen, device="cuda")).to(dtype))
    return x


def _rand(gen, shape, std, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def _quantise(x):
    """(whole numbers, step exponents) of rows in 32 bits; columns padded with zeros to whole blocks."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    v = torch.zeros(rows, blocks * BLOCK, dtype=torch.float32, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, blocks, BLOCK)
    bits = v.abs().amax(-1).view(torch.int32)          # of one block: NaN is carried by amax
    bad = bits >= 0x7F800000
    e = (((bits + 0x10000) >> 23) - 6).clamp(1, 254)   # the carry takes a largest value that would round to 128 up one step
    e = torch.where(bad, torch.full_like(e, 255), e)
    # times 2^(127-e), in two halves so that both are normal numbers
    up = 127 - e
    half = up // 2
    q = torch.round(v * torch.exp2(half.float()).unsqueeze(-1) * torch.exp2((up - half).float()).unsqueeze(-1))
    q = torch.where(bad.unsqueeze(-1), torch.zeros_like(q), q)
    return q.view(rows, blocks * BLOCK)[:, :cols], e


def _values(q, e):
    """What whole numbers and step exponents stand for, in 32 bits."""
    e = e.to(torch.int32)
    step = torch.where(e == 255, torch.full_like(e, 0x7FC00000), e << 23).view(torch.float32)
    return q.float() * step.repeat_interleave(BLOCK, 1)[:, : q.shape[1]]


def _kept(x):
    """A checkpoint in memory: rows of whole numbers and of exponents, both padded to 16 bytes."""
    q, e = _quantise(x.float())
    rows, cols = q.shape
    qs = torch.zeros(rows, -(-cols // 16) * 16, dtype=torch.int8, device=x.device)
    es = torch.ones(rows, -(-e.shape[1] // 16) * 16, dtype=torch.uint8, device=x.device)
    qs[:, :cols] = q.to(torch.int8)
    es[:, : e.shape[1]] = e.to(torch.uint8)
    return qs, es


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    s = {"c": c}
    if c["kind"] in ("norm", "norm8"):
        dt = DT[c.get("dtype", "bf16")]
        x = _stream_rows(gen, c["rows"], c["d"], c["pad"], dt)
        s["g"] = (1 + 0.2 * torch.randn(c["d"], generator=gen, device="cuda")).to(dt)
        s["b"] = _rand(gen, c["d"], 0.1, dt)
        if not c["bwd"]:
            s["x"] = x
            return s
        s["dy"] = _rand(gen, (c["rows"], c["d"]), 1e-3, dt)
        s["join"] = _rand(gen, (c["rows"], c["d"]), 1e-3, dt) if c["join"] else None
        # what the forward pass left: x and its statistics, or the normalised rows in 8 bits
        x32 = x.float()
        mean = x32.mean(1)
        x32 = x32 - mean.unsqueeze(1)
        s["rstd"] = torch.rsqrt(x32.square().mean(1) + EPS)
        if c["kind"] == "norm":
            s["x"], s["mean"] = x, mean
        else:
            s["q"], s["e"] = _kept(x32 * s["rstd"].unsqueeze(1))
        return s
    t, n, k = c["tokens"], c["n"], c["k"]
    if c["kind"] == "wgrad8":
        s["dy"] = _rand(gen, (t, n), 1e-3)
        if c["norm"]:
            s["q"], s["e"] = _kept(torch.randn(t, k, generator=gen, device="cuda"))   # normalised rows
            s["g"] = (1 + 0.2 * torch.randn(k, generator=gen, device="cuda")).bfloat16()
            s["b"] = _rand(gen, k, 0.1)
        else:
            x = _stream_rows(gen, t, k, 0, torch.bfloat16)
            if c["pack"]:
                s["x"] = x
            else:
                s["q"], s["e"] = _kept(x)
        s["base"] = _rand(gen, (n, k), 1e-2, torch.float32) if c["acc"] else None
        return s
    s["x"] = _rand(gen, (t, k), 1.0)
    s["w"] = _rand(gen, (n, k), 1.2 / math.sqrt(k))
    if c["kind"] == "linear":
        s["b"] = _rand(gen, n, 0.2) if c["bias"] else None
        s["res"] = _rand(gen, (t, n), 1.0) if c["res"] else None
    else:
        s["b"] = _rand(gen, n, 0.2)
        s["dy"] = _rand(gen, (t, k), 1e-3)
        s["w2"] = _rand(gen, (k, n), 1.0 / math.sqrt(n))
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from parameter_server_b200.ops import act8, linear, norm

    c = s["c"]
    kind = c["kind"]
    if kind == "norm":
        if not c["bwd"]:
            return norm.layer_norm(s["x"], s["g"], s["b"], EPS)
        return norm.layer_norm_backward(s["dy"], s["x"], s["g"], s["mean"], s["rstd"], residual_grad=s["join"])
    if kind == "norm8":
        if not c["bwd"]:
            y, x8, rstd = norm.layer_norm_act8(s["x"], s["g"], s["b"], EPS)
            return y, act8.act8_unpack(x8), rstd
        return norm.layer_norm_act8_backward(s["dy"], act8.Act8(s["q"], s["e"], c["d"]), s["g"], s["rstd"], residual_grad=s["join"])
    if kind == "linear":
        return linear.linear_act(s["x"], s["w"], s["b"], act=c["act"], residual=s["res"], save="bf16" if c["save"] else None)
    if kind == "mlp":
        y, h = linear.linear_act(s["x"], s["w"], s["b"], act=c["act"], save="act8" if c["bits"] == 8 else "bf16")
        return (y,) + linear.linear_act_dgrad(s["dy"], s["w2"], h, act=c["act"], recompute=True)
    x8 = act8.act8_pack(s["x"]) if c["pack"] else act8.Act8(s["q"], s["e"], c["k"])
    out = s["base"].clone() if c["acc"] else None
    if c["norm"]:
        db = linear.linear_bias_grad(s["dy"])
        return db, act8.act8_wgrad(s["dy"], x8, weight=s["g"], bias=s["b"], dy_sum=db, out=out, accumulate=c["acc"])
    return act8.act8_wgrad(s["dy"], x8, out=out, accumulate=c["acc"])


def _act(h, act):
    if act == "none":
        return h
    if act == "relu":
        return torch.where(h > 0, h, torch.zeros_like(h))
    if act == "gelu":
        return 0.5 * h * (1 + torch.erf(h * math.sqrt(0.5)))
    z = h if act == "silu" else 2 * math.sqrt(2 / math.pi) * (h + 0.044715 * h * h * h)   # (1 + tanh(u)) / 2 = 1 / (1 + exp(-2u))
    return h / (1 + torch.exp(-z))


def _act_slope(h, act):
    if act == "relu":
        return (h > 0).float()
    if act == "gelu":
        return 0.5 * (1 + torch.erf(h * math.sqrt(0.5))) + h * torch.exp(-0.5 * h * h) / math.sqrt(2 * math.pi)
    c = 2 * math.sqrt(2 / math.pi)
    z = h if act == "silu" else c * (h + 0.044715 * h * h * h)
    dz = 1.0 if act == "silu" else c * (1 + 3 * 0.044715 * h * h)
    s = 1 / (1 + torch.exp(-z))
    return s + h * s * (1 - s) * dz


def _norm_grads(xhat, dy, g, rstd, join):
    d = xhat.shape[1]
    p = dy * g
    dx = rstd.unsqueeze(1) * (p - p.sum(1, keepdim=True) / d - xhat * ((p * xhat).sum(1, keepdim=True) / d))
    if join is not None:
        dx = dx + join
    return dx, (dy * xhat).sum(0), dy.sum(0)


def _run_plain(s):
    c = s["c"]
    kind = c["kind"]
    if kind in ("norm", "norm8"):
        dt = s["g"].dtype
        g, b = s["g"].float(), s["b"].float()
        d = c["d"]
        if c["bwd"]:
            if kind == "norm":
                xhat = (s["x"].float() - s["mean"].unsqueeze(1)) * s["rstd"].unsqueeze(1)
            else:
                xhat = _values(s["q"][:, :d], s["e"][:, : -(-d // BLOCK)])
            dx, dw, db = _norm_grads(xhat, s["dy"].float(), g, s["rstd"], None if s["join"] is None else s["join"].float())
            return dx.to(dt), dw, db
        x = s["x"].float()
        mean = x.sum(1) / d
        cen = x - mean.unsqueeze(1)
        rstd = 1 / torch.sqrt((cen * cen).sum(1) / d + EPS)
        xhat = cen * rstd.unsqueeze(1)
        y = (xhat * g + b).to(dt)
        if kind == "norm":
            return y, mean, rstd
        return y, _values(*_quantise(xhat)).to(dt), rstd
    if kind == "wgrad8":
        x = _values(*_quantise(s["x"].float())) if c["pack"] else _values(s["q"][:, : c["k"]], s["e"][:, : -(-c["k"] // BLOCK)])
        if c["norm"]:
            x = x * s["g"].float() + s["b"].float()
        dy = s["dy"].float()
        dw = dy.t() @ x
        if c["acc"]:
            dw = s["base"] + dw
        return (dy.sum(0), dw) if c["norm"] else dw
    h = s["x"].float() @ s["w"].float().t()
    if s["b"] is not None:
        h = h + s["b"].float()
    y = _act(h, c["act"])
    if kind == "linear":
        if s["res"] is not None:
            y = y + s["res"].float()
        return (y.bfloat16(), h.bfloat16()) if c["save"] else y.bfloat16()
    kept = _values(*_quantise(h)) if c["bits"] == 8 else h.bfloat16().float()
    del h
    dh = (s["dy"].float() @ s["w2"].float()) * _act_slope(kept, c["act"])
    return y.bfloat16(), dh.bfloat16(), _act(kept, c["act"]).bfloat16()


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------

def _nearest8(x):
    """The values that an 8-bit checkpoint of rows in 64 bits stands for (finite rows)."""
    out = torch.empty_like(x)
    for j in range(0, x.shape[1], BLOCK):
        v = x[:, j:j + BLOCK]
        top = v.abs().amax(1, keepdim=True)
        _, ex = torch.frexp(top)                       # top = f 2^ex with f in [0.5, 1)
        step = torch.ldexp(torch.ones_like(top), ex - 7)
        step = torch.where(top / step >= 127.5, 2 * step, step)
        step = torch.clamp(step, min=2.0 ** -126)
        out[:, j:j + BLOCK] = torch.round(v / step) * step
    return out


def _stands_for(q, e, cols):
    """A checkpoint's values in 64 bits (finite blocks)."""
    return q[:, :cols].double() * torch.pow(2.0, e.double() - 127)[:, torch.arange(cols, device=q.device) // BLOCK]


def _phi(h, act, slope):
    """An activation in 64 bits, or its derivative."""
    if act == "none":
        return torch.ones_like(h) if slope else h
    if act == "relu":
        return (h > 0).double() if slope else h.clamp(min=0)
    if act == "gelu":
        cdf = torch.special.ndtr(h)
        return cdf + h * torch.exp(-h * h / 2) * (0.5 / math.pi) ** 0.5 if slope else h * cdf
    if act == "silu":
        s = torch.sigmoid(h)
        return s * (1 + h * (1 - s)) if slope else h * s
    a = (2 / math.pi) ** 0.5
    t = torch.tanh(a * (h + 0.044715 * h ** 3))
    return 0.5 * (1 + t) + 0.5 * h * (1 - t * t) * a * (1 + 0.134145 * h * h) if slope else 0.5 * h * (1 + t)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    kind = c["kind"]
    D = lambda t: None if t is None else t.double()  # noqa: E731
    if kind in ("norm", "norm8"):
        g, b = D(s["g"]), D(s["b"])
        if not c["bwd"]:
            x = D(s["x"])
            var, mean = torch.var_mean(x, 1, unbiased=False)
            rstd = (var + EPS) ** -0.5
            xhat = (x - mean[:, None]) * rstd[:, None]
            y = torch.addcmul(b, xhat, g)
            return (y, mean, rstd) if kind == "norm" else (y, _nearest8(xhat), rstd)
        rstd = D(s["rstd"])
        kept = (D(s["x"]) - D(s["mean"])[:, None]) * rstd[:, None] if kind == "norm" else _stands_for(s["q"], s["e"], c["d"])
        dy = D(s["dy"])
        p = dy * g
        dx = (p - p.mean(1, keepdim=True) - kept * (p * kept).mean(1, keepdim=True)) * rstd[:, None]
        if s["join"] is not None:
            dx += D(s["join"])
        return dx, torch.einsum("rd,rd->d", dy, kept), dy.sum(0)
    if kind == "wgrad8":
        if c["pack"]:
            x = _nearest8(D(s["x"]))
        else:
            x = _stands_for(s["q"], s["e"], c["k"])
        if c["norm"]:
            x = x * D(s["g"]) + D(s["b"])
        dy = D(s["dy"])
        dw = torch.mm(dy.t(), x)
        if c["acc"]:
            dw += D(s["base"])
        return (dy.sum(0), dw) if c["norm"] else dw
    h = torch.mm(D(s["x"]), D(s["w"]).t())
    if s["b"] is not None:
        h += D(s["b"])
    y = _phi(h, c["act"], False)
    if kind == "linear":
        if s["res"] is not None:
            y = y + D(s["res"])
        return (y, h) if c["save"] else y
    kept = _nearest8(h) if c["bits"] == 8 else h.bfloat16().double()   # what a later pass has is the checkpoint
    dh = torch.mm(D(s["dy"]), D(s["w2"])) * _phi(kept, c["act"], True)
    return y, dh, _phi(kept, c["act"], False)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    c = case
    kind = c["kind"]
    if kind in ("norm", "norm8"):
        rows, d = c["rows"], c["d"]
        el = rows * d
        size = 4 if c.get("dtype") == "f32" else 2
        join = size * el if c["join"] else 0
        kept8 = el + rows * -(-d // BLOCK)
        if not c["bwd"]:   # with 8 bits: the checkpoint is written, and read again for its values
            more = 2 * kept8 + size * el if kind == "norm8" else 0
            return {"bytes": 2 * size * el + more + 8 * rows + 2 * size * d, "flops": 8 * el}
        kept = kept8 + 4 * rows if kind == "norm8" else size * el + 8 * rows
        return {"bytes": kept + 2 * size * el + join + size * d + 8 * d, "flops": 14 * el}
    t, n, k = c["tokens"], c["n"], c["k"]
    if kind == "linear":
        out = 2 * t * n * (1 + int(c["res"]) + int(c["save"]))
        return {"bytes": 2 * (t * k + n * k) + (2 * n if c["bias"] else 0) + out, "flops": 2 * t * n * k}
    if kind == "mlp":   # x, w, y, checkpoint out; dy, w2, checkpoint in, dh and act(h) out
        kept = t * n + t * -(-n // BLOCK) if c["bits"] == 8 else 2 * t * n
        return {"bytes": 2 * (2 * t * k + 2 * n * k + 3 * t * n + n) + 2 * kept, "flops": 4 * t * n * k}
    kept = t * k + t * -(-k // BLOCK)
    pack = 2 * t * k + kept if c["pack"] else 0
    return {"bytes": 2 * t * n + kept + pack + 4 * n * k * (2 if c["acc"] else 1) + (4 * k + 4 * n if c["norm"] else 0), "flops": 2 * t * n * k}
