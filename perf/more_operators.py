"""The gated decoder block in training, as timed cases: the gated feed-forward layer, rotary positions, and dropout.

A case is a dict of plain values; ``prepare`` makes what a program holds before the call, ``run`` is one pass: the plain
form (elementary torch operations in 32 bits, rounded once at the end; angles in 64), or, where ``own`` is set, the calls into
the package. ``exact`` is the same in 64 bits, ``work`` what a pass cannot do without.

Kinds:

* ``glu``      act(x wg^T + bg) * (x wu^T + bu), with wg and wu the two halves of one weight [2F, K]. ``save``: both factors' values before
  the activation, [T, 2F], are returned too (16: in bf16; 0: not).
* ``glu_bwd``  the backward pass into them: with da = dy w2, the gradients da * u * act'(g) and da * act(g) side by side, and act(g) * u
  again for the weight gradient of the layer behind. ``bits``: g and u come in bf16 or as 8-bit checkpoints.
* ``rope``     rotary positions of queries and keys, forward or backward (``bwd``), out of place. ``layout``: "packed" (heads of q, k and v in
  one row of a QKV product), "heads" ([batch, heads, tokens, dim] in memory) or "rows" (tensors of their own). ``rot``: how many of
  a head's ``dim`` values turn; ``inter``: pairs are neighbours, not halves; ``scaling``: how frequencies were made longer.
* ``drop``     dropout with a mask that is formed from (seed, offset, row, column), with a residual (``res``), or its backward pass.
* ``drop_linear``  residual + dropout(x w^T + b).

The mask of dropout is Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) with counter
(column / 4, row, offset's low and high 32 bits) and key (seed's low and high 32 bits); a value is kept where word ``column % 4`` is at
least round(p * 2^32).

An 8-bit checkpoint holds 32 neighbours of a row as whole numbers of -127..127 and one power of two: the smallest step
2^(e-127), e in 1..249, at which the largest of them rounds to at most 127.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 32
BASE = 10000.0


def listed():
    return [
        # scoring one token: as fast as both projections' weights are read (d_model 2048, two thirds of the decoder's 8192 hidden values,
        # rounded up to a multiple of 128)
        dict(name="glu_1", kind="glu", tokens=1, f=5504, k=2048, act="silu", bias=False, save=0),
        # odd sizes, another activation, biases, and what the backward pass needs kept
        dict(name="glu_odd", kind="glu", tokens=1025, f=1000, k=776, act="gelu", bias=True, save=16),
        # one training micro-batch of the decoder: 8 sequences of 2048 tokens
        dict(name="glu_16k", kind="glu", tokens=16384, f=5504, k=2048, act="silu", bias=True, save=16),
        # backward for half a sequence
        dict(name="glu_bwd_1k", kind="glu_bwd", tokens=1024, f=5504, k=2048, act="silu", bits=16),
        # backward on the micro-batch from checkpoints in 8 bits
        dict(name="glu_bwd8_16k", kind="glu_bwd", tokens=16384, f=5504, k=2048, act="gelu_tanh", bits=8),
        # a single new token far into a long context
        dict(name="rope_1", kind="rope", batch=1, tokens=1, hq=16, hk=16, dim=128, rot=128, inter=False, layout="rows", dtype="bf16", bwd=False, scaling="yarn", first=131071),
        # the micro-batch's queries and keys as the QKV product left them
        dict(name="rope_16k", kind="rope", batch=8, tokens=2048, hq=16, hk=16, dim=128, rot=128, inter=False, layout="packed", dtype="bf16", bwd=False, scaling="none", first=0),
        # backward in 32 bits of a head that turns in part, neighbours paired, few key heads, odd sizes
        dict(name="rope_bwd_odd", kind="rope", batch=3, tokens=1001, hq=6, hk=2, dim=76, rot=50, inter=True, layout="heads", dtype="f32", bwd=True, scaling="linear", first=5),
        # the second half of 16 tokens' block: dropout on its way into the residual stream, where the launch is most of the time
        dict(name="drop_16", kind="drop", rows=16, cols=2048, dtype="bf16", pad=0, res=True, bwd=False, p=0.1),
        # the micro-batch's residual sum
        dict(name="drop_16k", kind="drop", rows=16384, cols=2048, dtype="bf16", pad=0, res=True, bwd=False, p=0.1),
        # backward of a model kept in 32 bits with an odd width and rows that are not packed
        dict(name="drop_bwd_odd", kind="drop", rows=4099, cols=1001, dtype="f32", pad=3, res=False, bwd=True, p=0.25),
        # attention's projection of the micro-batch, dropped out and added to the residual stream
        dict(name="drop_linear_16k", kind="drop_linear", tokens=16384, n=2048, k=2048, p=0.1),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    kind = rng.choice(["glu", "glu", "glu_bwd", "glu_bwd", "rope", "rope", "drop", "drop", "drop_linear"])
    acts = ["none", "relu", "gelu", "gelu_tanh", "silu"]
    if kind in ("glu", "glu_bwd"):
        f, k = log(64, 8192), log(128, 8192)
        if rng.random() < 0.7:
            f, k = -(-f // 8) * 8, -(-k // 8) * 8
        tokens = log(1, max(1, min(16384, 16384 * 5504 * 2048 // (f * k))))
        if kind == "glu":
            return dict(kind=kind, tokens=tokens, f=f, k=k, act=rng.choice(acts), bias=rng.random() < 0.5, save=rng.choice([0, 16]))
        return dict(kind=kind, tokens=tokens, f=f, k=k, act=rng.choice(acts), bits=rng.choice([16, 8]))
    if kind == "rope":
        dim = rng.choice([32, 64, 80, 96, 128, 128, 192, 256]) if rng.random() < 0.8 else 2 * log(4, 150)
        rot = dim if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2)
        hq = log(1, 64)
        hk = max(1, hq // rng.choice([1, 1, 2, 4, 8]))
        batch = log(1, 16)
        tokens = log(1, max(1, 16384 * 32 * 128 // (batch * (hq + hk) * dim)))
        return dict(kind=kind, batch=batch, tokens=tokens, hq=hq, hk=hk, dim=dim, rot=rot, inter=rng.random() < 0.4, layout=rng.choice(["packed", "heads", "rows"]),
                    dtype=rng.choice(["bf16", "bf16", "f32"]), bwd=rng.random() < 0.4, scaling=rng.choice(["none", "linear", "ntk", "yarn"]), first=rng.choice([0, 0, log(1, 1 << 20)]))
    p = rng.choice([0.0, 0.05, 0.1, 0.3, 0.5, round(rng.uniform(0.01, 0.9), 3)])
    if kind == "drop":
        cols = log(16, 16384)
        rows = log(1, max(1, min(100000, 16384 * 2048 // cols)))
        bwd = rng.random() < 0.4
        return dict(kind=kind, rows=rows, cols=cols, dtype=rng.choice(["bf16", "bf16", "f32"]), pad=rng.choice([0, 0, 5, 8]), res=not bwd and rng.random() < 0.7, bwd=bwd, p=p)
    n, k = log(128, 8192), log(128, 8192)
    if rng.random() < 0.7:
        n, k = -(-n // 8) * 8, -(-k // 8) * 8
    return dict(kind=kind, tokens=log(1, max(1, min(16384, 16384 * 2048 * 2048 // (n * k)))), n=n, k=k, p=p)


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _rand(gen, shape, std, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


def _quantise(x):
    """(whole numbers, step exponents) of finite rows in 32 bits; columns padded with zeros to whole blocks."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    v = torch.zeros(rows, blocks * BLOCK, dtype=torch.float32, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, blocks, BLOCK)
    bits = v.abs().amax(-1).view(torch.int32)
    e = (((bits + 0x10000) >> 23) - 6).clamp(1, 254)   # the carry takes a largest value that would round to 128 up one step
    q = torch.round(v * torch.exp2(127.0 - e.float()).unsqueeze(-1))
    return q.view(rows, blocks * BLOCK)[:, :cols], e


def _kept(x):
    """A checkpoint in memory: rows of whole numbers and of exponents, both padded to 16 bytes."""
    q, e = _quantise(x.float())
    rows, cols = q.shape
    qs = torch.zeros(rows, -(-cols // 16) * 16, dtype=torch.int8, device=x.device)
    es = torch.ones(rows, -(-e.shape[1] // 16) * 16, dtype=torch.uint8, device=x.device)
    qs[:, :cols] = q.to(torch.int8)
    es[:, : e.shape[1]] = e.to(torch.uint8)
    return qs, es


def _frequencies(rot, scaling):
    """(radians per position of each pair, in 64 bits; the factor on cosine and sine), for contexts four times as long as the 4096
    positions that a model was trained on."""
    i = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda")
    factor, trained = 4.0, 4096
    if scaling == "ntk" and rot > 2:
        return (BASE * factor ** (rot / (rot - 2))) ** (-i / rot), 1.0
    freqs = BASE ** (-i / rot)
    if scaling in ("linear", "ntk"):   # (a single pair has nothing to spread the stretch over)
        return freqs / factor, 1.0
    if scaling == "yarn":   # pairs that turn more than 32 times over the trained length stay, those below one turn are stretched
        kept = ((freqs * trained / (2 * math.pi) - 1) / (32 - 1)).clamp(0, 1)
        return freqs * kept + freqs / factor * (1 - kept), 0.1 * math.log(factor) + 1
    return freqs, 1.0


def _heads(gen, c, heads, std):
    """Queries or keys as [batch, tokens, heads, dim] in the case's layout ("packed" is made for q and k together)."""
    dt = DT[c["dtype"]]
    if c["layout"] == "heads":
        return _rand(gen, (c["batch"], heads, c["tokens"], c["dim"]), std, dt).transpose(1, 2)
    return _rand(gen, (c["batch"], c["tokens"], heads, c["dim"]), std, dt)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 29)
    s = {"c": c}
    kind = c["kind"]
    if kind == "rope":
        std = 1e-3 if c["bwd"] else 1.0
        if c["layout"] == "packed":
            qkv = _heads(gen, c, c["hq"] + 2 * c["hk"], std)
            s["q"], s["k"] = qkv[:, :, :c["hq"]], qkv[:, :, c["hq"]:c["hq"] + c["hk"]]
        else:
            s["q"], s["k"] = _heads(gen, c, c["hq"], std), _heads(gen, c, c["hk"], std)
        s["freqs"], s["scale"] = _frequencies(c["rot"], c["scaling"])
        # every sequence of the batch at a place of its own, as after left padding
        start = c["first"] + torch.randint(0, 1 + c["first"] // 8, (c["batch"], 1), generator=gen, device="cuda")
        s["pos"] = start + torch.arange(c["tokens"], device="cuda")
        return s
    if kind in ("drop", "drop_linear"):
        s["seed"], s["offset"] = (int(seed) * 0x9E3779B97F4A7C15 + 0x1234567) % (1 << 63), int(seed) % 1000 * (1 << 30) + 7
    if kind == "drop":
        dt = DT[c["dtype"]]
        x = _rand(gen, (c["rows"], c["cols"] + c["pad"]), 1e-3 if c["bwd"] else 1.0, dt)[:, :c["cols"]]
        s["x"] = x
        s["res"] = _rand(gen, (c["rows"], c["cols"]), 2.0, dt) if c["res"] else None
        return s
    t, k = c["tokens"], c["k"]
    if kind == "drop_linear":
        s["x"], s["w"], s["b"] = _rand(gen, (t, k), 1.0), _rand(gen, (c["n"], k), 1.2 / math.sqrt(k)), _rand(gen, c["n"], 0.2)
        s["res"] = _rand(gen, (t, c["n"]), 2.0)
        return s
    f = c["f"]
    if kind == "glu":
        s["x"], s["w"] = _rand(gen, (t, k), 1.0), _rand(gen, (2 * f, k), 1.2 / math.sqrt(k))
        s["b"] = _rand(gen, 2 * f, 0.2) if c["bias"] else None
        return s
    s["dy"], s["w2"] = _rand(gen, (t, k), 1e-3), _rand(gen, (k, f), 1.0 / math.sqrt(f))
    if c["bits"] == 16:
        s["h"] = _rand(gen, (t, 2 * f), 1.2)
    else:
        s["g8"], s["u8"] = _kept(_rand(gen, (t, f), 1.2)), _kept(_rand(gen, (t, f), 1.2))
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from parameter_server_b200.ops import act8, dropout, gated, linear, rotary

    c = s["c"]
    kind = c["kind"]
    if kind == "glu":
        return gated.gated_linear(s["x"], s["w"], s["b"], act=c["act"], save="bf16" if c["save"] else None)
    if kind == "glu_bwd":
        h = s["h"] if c["bits"] == 16 else (act8.Act8(*s["g8"], c["f"]), act8.Act8(*s["u8"], c["f"]))
        return gated.gated_linear_dgrad(s["dy"], s["w2"], h, act=c["act"], recompute=True)
    if kind == "rope":
        call = rotary.rotary_backward if c["bwd"] else rotary.rotary
        return call(s["q"], s["k"], s["freqs"], s["pos"], interleaved=c["inter"], scale=s["scale"])
    if kind == "drop":
        if c["bwd"]:
            return dropout.dropout_backward(s["x"], c["p"], s["seed"], s["offset"])
        return dropout.dropout(s["x"], c["p"], s["seed"], s["offset"], residual=s["res"])
    return linear.linear_act(s["x"], s["w"], s["b"], residual=s["res"], dropout=(c["p"], s["seed"], s["offset"]))


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
    if act == "none":
        return torch.ones_like(h)
    if act == "relu":
        return (h > 0).float()
    if act == "gelu":
        return 0.5 * (1 + torch.erf(h * math.sqrt(0.5))) + h * torch.exp(-0.5 * h * h) / math.sqrt(2 * math.pi)
    c = 2 * math.sqrt(2 / math.pi)
    z = h if act == "silu" else c * (h + 0.044715 * h * h * h)
    dz = 1.0 if act == "silu" else c * (1 + 3 * 0.044715 * h * h)
    s = 1 / (1 + torch.exp(-z))
    return s + h * s * (1 - s) * dz


def _turned(x, freqs, pos, scale, inter, back):
    """Queries or keys [batch, tokens, heads, dim] with their first 2 * len(freqs) values turned."""
    angle = pos.double().unsqueeze(-1) * freqs            # 32 bits lose the angles of far positions
    cos, sin = (torch.cos(angle) * scale).float().unsqueeze(2), (torch.sin(angle) * scale).float().unsqueeze(2)
    if back:
        sin = -sin
    y = x.float()
    rot = 2 * freqs.numel()
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if inter else (y[..., : rot // 2], y[..., rot // 2:rot])
    first, second = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((first, second), -1).flatten(-2) if inter else torch.cat((first, second), -1)
    return torch.cat((turned, y[..., rot:]), -1).to(x.dtype)


LOW = 0xFFFFFFFF


def _keep(rows, cols, p, seed, offset, device):
    """The mask of dropout. Words of 32 bits are held in 64: a product's low and high word are its bits, whether it wrapped or not."""
    g, r = torch.arange(-(-cols // 4), device=device), torch.arange(rows, device=device)
    c0, c1 = g.expand(rows, -1), r.unsqueeze(1).expand(-1, g.numel())
    c2, c3 = torch.full_like(c0, offset & LOW), torch.full_like(c0, offset >> 32 & LOW)
    k0, k1 = seed & LOW, seed >> 32 & LOW
    for _ in range(10):   # the generator's rounds
        m0, m1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = m1 >> 32 & LOW ^ c1 ^ k0, m1 & LOW, m0 >> 32 & LOW ^ c3 ^ k1, m0 & LOW
        k0, k1 = k0 + 0x9E3779B9 & LOW, k1 + 0xBB67AE85 & LOW
    return torch.stack((c0, c1, c2, c3), -1).flatten(1)[:, :cols] >= int(p * 2.0 ** 32 + 0.5)


def _dropped(x, p, seed, offset):
    """Dropout of rows in 32 bits. What is kept grows by the share of words that keep a value."""
    scale = 2.0 ** 32 / (2 ** 32 - int(p * 2.0 ** 32 + 0.5))
    return torch.where(_keep(x.shape[0], x.shape[1], p, seed, offset, x.device), x * scale, torch.zeros_like(x))


def _run_plain(s):
    c = s["c"]
    kind = c["kind"]
    if kind == "glu":
        h = s["x"].float() @ s["w"].float().t()
        if s["b"] is not None:
            h = h + s["b"].float()
        y = (_act(h[:, : c["f"]], c["act"]) * h[:, c["f"]:]).bfloat16()
        return (y, h.bfloat16()) if c["save"] else y
    if kind == "glu_bwd":
        f = c["f"]
        if c["bits"] == 16:
            g, u = s["h"][:, :f].float(), s["h"][:, f:].float()
        else:
            g, u = (q[:, :f].float() * torch.exp2(e.float() - 127).repeat_interleave(BLOCK, 1)[:, :f] for q, e in (s["g8"], s["u8"]))
        da = s["dy"].float() @ s["w2"].float()
        a = _act(g, c["act"])
        return torch.cat((da * u * _act_slope(g, c["act"]), da * a), 1).bfloat16(), (a * u).bfloat16()
    if kind == "rope":
        more = (s["freqs"], s["pos"], s["scale"], c["inter"], c["bwd"])
        return _turned(s["q"], *more), _turned(s["k"], *more)
    if kind == "drop":
        y = _dropped(s["x"].float(), c["p"], s["seed"], s["offset"])
        return (y if s["res"] is None else y + s["res"].float()).to(s["x"].dtype)
    y = s["x"].float() @ s["w"].float().t() + s["b"].float()
    return (_dropped(y, c["p"], s["seed"], s["offset"]) + s["res"].float()).bfloat16()


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------

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


def _stands_for(q, e, cols):
    """A checkpoint's values in 64 bits (finite blocks)."""
    return q[:, :cols].double() * torch.pow(2.0, e.double() - 127)[:, torch.arange(cols, device=q.device) // BLOCK]


def _times(a, m):
    """(high, low) words of the product of 32-bit words and a constant, by halves of 16 bits."""
    al, ah, ml, mh = a & 0xFFFF, a >> 16, m & 0xFFFF, m >> 16
    mid = al * mh + (al * ml >> 16)
    cross = ah * ml + (mid & 0xFFFF)
    return ah * mh + (mid >> 16) + (cross >> 16), (cross & 0xFFFF) << 16 | al * ml & 0xFFFF


def _mask64(rows, cols, p, seed, offset, device):
    col = torch.arange((cols + 3) // 4 * 4, device=device)
    group = (col // 4)[::4].repeat(rows, 1)
    x = [group, torch.arange(rows, device=device)[:, None] + 0 * group, 0 * group + offset % 2 ** 32, 0 * group + offset // 2 ** 32 % 2 ** 32]
    key = [seed % 2 ** 32, seed // 2 ** 32 % 2 ** 32]
    for n in range(10):
        (ha, la), (hb, lb) = _times(x[0], 0xD2511F53), _times(x[2], 0xCD9E8D57)
        x = [hb ^ x[1] ^ (key[0] + n * 0x9E3779B9) % 2 ** 32, lb, ha ^ x[3] ^ (key[1] + n * 0xBB67AE85) % 2 ** 32, la]
    words = torch.empty(rows, col.numel(), dtype=torch.int64, device=device)
    for j in range(4):
        words[:, j::4] = x[j]
    return words[:, :cols] >= math.floor(p * 2.0 ** 32 + 0.5)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    kind = c["kind"]
    D = lambda t: None if t is None else t.double()  # noqa: E731
    if kind == "glu":
        h = torch.mm(D(s["x"]), D(s["w"]).t())
        if s["b"] is not None:
            h += D(s["b"])
        g, u = h.split(c["f"], 1)
        y = _phi(g, c["act"], False) * u
        return (y, h) if c["save"] else y
    if kind == "glu_bwd":
        g, u = D(s["h"]).split(c["f"], 1) if c["bits"] == 16 else (_stands_for(*s["g8"], c["f"]), _stands_for(*s["u8"], c["f"]))
        da = torch.mm(D(s["dy"]), D(s["w2"]))
        act = _phi(g, c["act"], False)
        dh = torch.empty(g.shape[0], 2 * c["f"], dtype=torch.float64, device=g.device)
        dh[:, : c["f"]] = _phi(g, c["act"], True).mul_(da).mul_(u)
        dh[:, c["f"]:] = da.mul_(act)
        return dh, act * u
    if kind == "rope":
        angle = torch.einsum("bt,i->bti", D(s["pos"]), s["freqs"])
        turn = torch.polar(torch.full_like(angle, s["scale"]), -angle if c["bwd"] else angle)[:, :, None]
        outs = []
        for x in (D(s["q"]), D(s["k"])):
            out = x.contiguous().clone()
            part = x[..., : c["rot"]].reshape(*x.shape[:3], *((-1, 2) if c["inter"] else (2, -1)))
            if not c["inter"]:
                part = part.transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn)
            out[..., : c["rot"]] = (z if c["inter"] else z.transpose(-1, -2)).reshape(*x.shape[:3], c["rot"])
            outs.append(out)
        return tuple(outs)
    if kind == "drop":
        x = D(s["x"])
    else:
        x = torch.addmm(D(s["b"]), D(s["x"]), D(s["w"]).t())
    kept = _mask64(x.shape[0], x.shape[1], c["p"], s["seed"], s["offset"], x.device)
    x = x.masked_fill(~kept, 0.0) / (1 - math.floor(c["p"] * 2.0 ** 32 + 0.5) / 2.0 ** 32)
    return x if s["res"] is None else x + D(s["res"])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    c = case
    kind = c["kind"]
    if kind == "rope":
        rows = c["batch"] * c["tokens"]
        el = rows * (c["hq"] + c["hk"]) * c["dim"]
        return {"bytes": 2 * el * (4 if c["dtype"] == "f32" else 2) + 8 * rows + 4 * c["rot"], "flops": 3 * rows * (c["hq"] + c["hk"]) * c["rot"]}
    if kind == "drop":
        el = c["rows"] * c["cols"]
        return {"bytes": el * (4 if c["dtype"] == "f32" else 2) * (3 if c["res"] else 2), "flops": 15 * el}
    t, k = c["tokens"], c["k"]
    if kind == "drop_linear":
        return {"bytes": 2 * (t * k + c["n"] * k + c["n"] + 2 * t * c["n"]), "flops": 2 * t * c["n"] * k}
    f = c["f"]
    if kind == "glu":
        return {"bytes": 2 * (t * k + 2 * f * k + t * f) + (4 * f if c["bias"] else 0) + (4 * t * f if c["save"] else 0), "flops": 4 * t * f * k}
    kept = 4 * t * f if c["bits"] == 16 else 2 * (t * f + t * -(-f // BLOCK))
    return {"bytes": 2 * (t * k + f * k) + kept + 6 * t * f, "flops": 2 * t * f * k}
