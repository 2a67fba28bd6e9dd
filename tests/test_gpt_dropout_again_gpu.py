"""A decoder with dropout whose passes are run again: by recomputation inside a backward pass."""
import pytest
import torch
from test_gpt_fused_autograd_gpu import SIZES, batch, close, grads, once
from torch.utils.checkpoint import checkpoint

from parameter_server_b200.models.gpt import GPT, GPTConfig

pytestmark = pytest.mark.gpu
PARTS = [dict(dropout=0.1), dict(gated=True, rotary=True, dropout=0.3)]


def model_of(bits, parts):
    return GPT(GPTConfig(**SIZES, **parts, fused=True, act_bits=bits), seed=1)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("parts", PARTS)
def test_recomputation_draws_the_same_masks(parts, bits):
    model = model_of(bits, parts)
    loss0, one = once(model)
    other, tokens, targets = model_of(bits, parts), *batch()
    other.zero_grads()
    loss = checkpoint(lambda t: other.forward(t, targets)[1], tokens, use_reentrant=False)
    loss.backward()
    assert loss.item() == loss0
    close(grads(other), one)
    assert other.drop_passes == model.drop_passes == 1
    other.check()


@pytest.mark.parametrize("parts", PARTS)
def test_each_of_several_passes_finds_its_own(parts):
    """Two passes before one backward pass, which runs them again in the other order."""
    model, other = model_of(16, parts), model_of(16, parts)
    tokens, targets = batch()
    for m in (model, other):
        m.zero_grads()
    halves = [(t, g) for t, g in zip(tokens.chunk(2), targets.chunk(2))]
    plain = [model.forward(t, g)[1] for t, g in halves]
    again = [checkpoint(lambda t, g=g: other.forward(t, g)[1], t, use_reentrant=False) for t, g in halves]
    sum(plain).backward()
    sum(again).backward()
    assert [p.item() for p in plain] == [p.item() for p in again]
    close(grads(other), grads(model))
    assert other.drop_passes == model.drop_passes == 2
    # the pass behind them draws anew, as without recomputation
    assert once(other)[0] == once(model)[0]


def test_a_graph_of_recomputed_passes_may_be_run_twice():
    model, other = model_of(8, PARTS[1]), model_of(8, PARTS[1])
    tokens, targets = batch()
    _, one = once(model)
    other.zero_grads()
    loss = checkpoint(lambda t: other.forward(t, targets)[1], tokens, use_reentrant=False)
    loss.backward(retain_graph=True)
    loss.backward()
    close(grads(other), one, 2.0)
    assert other.drop_passes == 1


def test_recomputation_that_cannot_know_its_masks_is_refused():
    """Without torch's generators put back, or where the first run was one without gradients and dropped nothing."""
    tokens, targets = batch()
    model = model_of(16, PARTS[0])
    loss = checkpoint(lambda t: model.forward(t, targets)[1], tokens, use_reentrant=False, preserve_rng_state=False)
    with pytest.raises(RuntimeError, match="recomput"):
        loss.backward()
    del loss
    model = model_of(16, PARTS[0])
    leaf = torch.ones((), device="cuda", requires_grad=True)
    loss = checkpoint(lambda one: model.forward(tokens, targets)[1] * one, leaf, use_reentrant=True)
    with pytest.raises(RuntimeError, match="recomput"):
        loss.backward()
    torch.cuda.synchronize()
