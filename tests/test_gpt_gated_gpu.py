"""The decoder with a gated hidden layer, rotary positions and dropout: its loss and gradients against the same decoder in torch operations in 32 bits
with the same masks; what it keeps, and what it refuses."""
import math

import philox64
import pytest
import torch
import torch.nn.functional as F

from parameter_server_b200.models.gpt import GPT, GPTConfig

SIZES = dict(n_layer=2, d_model=256, n_head=4, d_ff=680, vocab=512, seq_len=64, lr=3e-3, weight_decay=0.0, fused=True)
gpu = pytest.mark.gpu


def batch():
    data = torch.randint(0, 512, (8, 65), generator=torch.Generator().manual_seed(0)).cuda()
    return data[:, :-1], data[:, 1:]


def grads_of(model, tokens, targets):
    model.zero_grads()
    _, loss = model.forward(tokens, targets)
    loss.backward()
    for name, p in model._leaves.items():
        if p.grad is not None:
            model.main.grads[name].add_(p.grad.float())
    torch.cuda.synchronize()
    return loss.item(), {k: v.clone() for k, v in model.main.grads.items()}


def reference(model, tokens, targets, passes):
    """(loss, gradients) by torch's own operations; ``passes``: how many passes with dropout the model has had."""
    cfg = model.cfg
    P = {k: v.detach().float().requires_grad_(True) for k, v in model.main.params.items()}
    B, T = tokens.shape
    d, H = cfg.d_model, cfg.n_head

    def drop(x, site):
        if not cfg.dropout:
            return x
        mask = torch.from_numpy(philox64.kept(B * T, d, cfg.dropout, model.drop_seed, (passes << 16) + site)).cuda()
        return torch.where(mask, x.reshape(B * T, d) * philox64.grown(cfg.dropout), 0.0).view(B, T, d)

    def turn(x):   # [B, T, H, hd], halves
        half = d // H // 2
        angle = torch.arange(T, device="cuda").double()[:, None] * cfg.rotary_base ** (-torch.arange(half, device="cuda").double() / half)
        c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
        return torch.cat((x[..., :half] * c - x[..., half:] * s, x[..., :half] * s + x[..., half:] * c), -1)

    x = F.embedding(tokens, P["wte"])
    if not cfg.rotary:
        x = x + P["wpe"][:T]
    x = drop(x, 2 * cfg.n_layer)
    for i in range(cfg.n_layer):
        y = F.layer_norm(x, (d,), P[f"h{i}.ln1.g"], P[f"h{i}.ln1.b"])
        q, k, v = (y @ P[f"h{i}.qkv.w"].t() + P[f"h{i}.qkv.b"]).view(B, T, 3, H, d // H).unbind(2)
        if cfg.rotary:
            q, k = turn(q), turn(k)
        a = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=True).transpose(1, 2).reshape(B, T, d)
        x = x + drop(a @ P[f"h{i}.proj.w"].t() + P[f"h{i}.proj.b"], 2 * i)
        y = F.layer_norm(x, (d,), P[f"h{i}.ln2.g"], P[f"h{i}.ln2.b"])
        h = y @ P[f"h{i}.fc.w"].t() + P[f"h{i}.fc.b"]
        f = F.silu(h[..., :cfg.d_ff]) * h[..., cfg.d_ff:] if cfg.gated else F.gelu(h, approximate="tanh")
        x = x + drop(f @ P[f"h{i}.out.w"].t() + P[f"h{i}.out.b"], 2 * i + 1)
    x = F.layer_norm(x, (d,), P["lnf.g"], P["lnf.b"])
    loss = F.cross_entropy((x @ P["wte"].t()).view(-1, cfg.vocab), targets.reshape(-1))
    loss.backward()
    return loss.item(), {k: v.grad for k, v in P.items()}


# One rounding of 2^-9 per bf16 tensor on the way, about ten deep: a few percent of a gradient in norm; 8-bit checkpoints add about 1 % of a
# block's values each (the bounds of the fused decoder's other tests).
@gpu
@pytest.mark.parametrize("bits,limit", [(16, 0.05), (8, 0.08)])
@pytest.mark.parametrize("parts", [dict(gated=True), dict(rotary=True), dict(dropout=0.2), dict(gated=True, rotary=True, rotary_base=500.0, dropout=0.1)])
def test_loss_and_gradients(parts, bits, limit):
    model = GPT(GPTConfig(**SIZES, **parts, act_bits=bits), seed=1)
    tokens, targets = batch()
    for passes in range(2):   # the second pass draws anew
        loss, grads = grads_of(model, tokens, targets)
        want, wanted = reference(model, tokens, targets, passes)
        model.check()
        assert abs(loss - want) < 1e-2
        assert set(grads) == set(wanted)
        for name in grads:
            off = (grads[name] - wanted[name]).norm() / wanted[name].norm().clamp_min(1e-12)
            assert off < limit, (name, off.item())


@gpu
@pytest.mark.parametrize("bits", [16, 8])
def test_a_graph_may_be_run_twice_and_steps_run(bits):
    model = GPT(GPTConfig(**SIZES, gated=True, rotary=True, dropout=0.1, act_bits=bits), seed=2)
    tokens, targets = batch()
    model.zero_grads()
    _, loss = model.forward(tokens, targets)
    loss.backward(retain_graph=True)
    once = {k: v.clone() for k, v in model.main.grads.items()}
    loss.backward()
    for name, g in model.main.grads.items():
        assert torch.allclose(g, 2 * once[name], rtol=1e-5, atol=1e-8), name
    before = model.main.params["h0.fc.w"].clone()
    for _ in range(3):
        assert math.isfinite(model.train_step(tokens, targets, micro_batches=2).item())
    model.check()
    assert model.drop_passes == 7 and not torch.equal(before, model.main.params["h0.fc.w"])


@gpu
def test_nothing_is_dropped_where_nothing_is_trained():
    model, same = (GPT(GPTConfig(**SIZES, gated=True, rotary=True, dropout=p), seed=3) for p in (0.5, 0.0))
    tokens, targets = batch()
    with torch.no_grad():
        assert torch.equal(model.forward(tokens, targets)[1], same.forward(tokens, targets)[1])
    assert torch.equal(model.forward(tokens)[0], same.forward(tokens)[0]) and model.drop_passes == 0
    assert not torch.equal(model.forward(tokens, targets)[1], same.forward(tokens, targets)[1])


@gpu
@pytest.mark.parametrize("bits", [16, 8])
def test_what_a_gated_layer_keeps(bits):
    """Per token and layer: the values before the activation of both factors, in 16 bits or in 8 and a byte per 32."""
    D, HIDDEN, SEQ, BATCH = 512, 1344, 1024, 4
    tokens = torch.randint(0, 512, (BATCH, SEQ), generator=torch.Generator().manual_seed(0)).cuda()

    def held(layers):
        model = GPT(GPTConfig(n_layer=layers, d_model=D, n_head=8, d_ff=HIDDEN, vocab=512, seq_len=SEQ, fused=True, gated=True, rotary=True, dropout=0.1, act_bits=bits), seed=1)
        _, loss = model.forward(tokens, tokens)
        loss.backward()
        del loss
        torch.cuda.synchronize()
        before = torch.cuda.memory_stats()["requested_bytes.all.current"]
        _, loss = model.forward(tokens, tokens)
        torch.cuda.synchronize()
        return torch.cuda.memory_stats()["requested_bytes.all.current"] - before

    attention = 2 * 4 * D + 4 * 8
    if bits == 8:
        rest = 2 * (D + D // 32 + 4) + 2 * (HIDDEN + 48)   # (rows of exponents are padded to 16)
    else:
        rest = 2 * (2 * 2 * D + 8) + 4 * HIDDEN
    assert (held(4) - held(2)) / 2 / (BATCH * SEQ) <= 1.02 * (attention + rest)


def test_parts_need_the_fused_blocks():
    for parts in (dict(gated=True), dict(rotary=True), dict(dropout=0.1)):
        with pytest.raises(ValueError, match="fused"):
            GPT(GPTConfig(**{**SIZES, "fused": False}, **parts), device="cpu")
    for p in (1.0, -0.1, 2.0):
        with pytest.raises(ValueError, match="dropout"):
            GPT(GPTConfig(**SIZES, dropout=p), device="cpu")
    with pytest.raises(ValueError, match="rotary"):
        GPT(GPTConfig(**{**SIZES, "d_model": 252, "n_head": 12}, rotary=True), device="cpu")


def test_parameters_are_counted():
    d, f = 2048, 5504
    cfg = GPTConfig(d_ff=f, gated=True, rotary=True, fused=True)
    assert cfg.n_params() == 50304 * d + 24 * (4 * d * d + 3 * d * f + 9 * d + 2 * f) + 2 * d
    assert GPTConfig().n_params() == 50304 * d + 2048 * d + 24 * (4 * d * d + 2 * d * 8192 + 9 * d + 8192) + 2 * d
