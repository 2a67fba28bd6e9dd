"""A fused decoder under autograd's own tools: a graph that is run twice, hooks on what is saved, changes in place, recomputation; and
with its QKV weights in tables of their own, as several ranks have them."""
import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks
from torch.utils.checkpoint import checkpoint

from parameter_server_b200.models.gpt import GPT, GPTConfig
from parameter_server_b200.ops.dense import DenseTable

pytestmark = pytest.mark.gpu

SIZES = dict(n_layer=2, d_model=256, n_head=4, d_ff=1024, vocab=512, seq_len=64, lr=3e-3, weight_decay=0.0)


def model_of(bits):
    return GPT(GPTConfig(**SIZES, fused=True, act_bits=bits), seed=1)


def batch():
    data = torch.randint(0, 512, (8, 65), generator=torch.Generator().manual_seed(0)).cuda()
    return data[:, :-1], data[:, 1:]


def grads(model):
    torch.cuda.synchronize()
    return {k: v.clone() for k, v in model.main.grads.items()}


def close(a, b, scale=1.0):
    """The same sums in another order (attention's backward pass adds with atomics): bf16 values on the way round the other way."""
    for name in a:
        off = (a[name] - scale * b[name]).norm() / b[name].norm().clamp_min(1e-12)
        assert off <= 0.01, (name, off.item())


def once(model):
    model.zero_grads()
    _, loss = model.forward(*batch())
    loss.backward()
    return loss.item(), grads(model)


@pytest.mark.parametrize("bits", [16, 8])
def test_a_retained_graph_runs_twice(bits):
    model = model_of(bits)
    _, one = once(model)
    model.zero_grads()
    _, loss = model.forward(*batch())
    loss.backward(retain_graph=True)
    loss.backward()
    close(grads(model), one, 2.0)   # gradients of the blocks add up in the dense table
    model.check()


@pytest.mark.parametrize("bits", [16, 8])
def test_hooks_see_everything_that_is_saved(bits):
    model = model_of(bits)
    loss0, one = once(model)
    with save_on_cpu():
        loss1, two = once(model)
    assert loss1 == loss0
    close(two, one)
    # a block's norms and hidden layer are among what is saved: 8 bits as they are, 16 bits as bf16
    seen = []
    with saved_tensors_hooks(lambda t: seen.append((tuple(t.shape), t.dtype)) or t, lambda t: t):
        model.forward(*batch())
    tokens, d, hidden = 8 * 64, SIZES["d_model"], SIZES["d_ff"]
    kept = torch.int8 if bits == 8 else torch.bfloat16
    assert seen.count(((tokens, hidden), kept)) == SIZES["n_layer"]
    assert seen.count(((tokens, d), kept)) >= 2 * SIZES["n_layer"]
    model.check()


@pytest.mark.parametrize("bits", [16, 8])
def test_a_change_in_place_is_noticed(bits):
    model = model_of(bits)
    _, loss = model.forward(*batch())
    with torch.no_grad():
        model.main.params["h0.fc.w"].mul_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("bits", [16, 8])
def test_recomputation_gives_the_same(bits):
    model = model_of(bits)
    loss0, one = once(model)
    model.zero_grads()
    tokens, targets = batch()
    loss = checkpoint(lambda t: model.forward(t, targets)[1], tokens, use_reentrant=False)
    loss.backward()
    assert loss.item() == loss0
    close(grads(model), one)
    model.check()


@pytest.mark.parametrize("bits", [16, 8])
def test_qkv_weights_in_tables_of_their_own(bits):
    """What a model on several ranks does with the tables whose rows it gathers in the product, on one rank, which has all rows."""
    model = model_of(bits)
    loss0, one = once(model)
    d = SIZES["d_model"]
    for i in range(SIZES["n_layer"]):
        table = DenseTable({"w": (3 * d, d)}, "adamw", dict(lr=SIZES["lr"]), grad_dtype=torch.float32, device=model.device, scatter_peers=False)
        table.load({"w": model.main.params[f"h{i}.qkv.w"].detach().float().cpu()})
        table.zero_grads()
        model.qkv[i] = table
    model.zero_grads()
    _, loss = model.forward(*batch())
    loss.backward()
    two = grads(model)
    for i in range(SIZES["n_layer"]):
        assert (two[f"h{i}.qkv.w"] == 0).all()
        two[f"h{i}.qkv.w"] = model.qkv[i].grads["w"].clone()
    close(two, one)
    assert abs(loss.item() - loss0) < 2e-3   # the product itself is another kernel's
    model.check()
