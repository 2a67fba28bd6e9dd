"""Which masks a pass of the decoder draws: every pass new ones, a recomputed one its own, every rank others."""
import gc

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from parameter_server_b200.models.gpt import GPT, GPTConfig

SIZES = dict(n_layer=2, d_model=32, n_head=4, d_ff=40, vocab=64, seq_len=16, fused=True, dropout=0.1)


def model_of(seed=3):
    return GPT(GPTConfig(**SIZES), device="cpu", seed=seed)


class Scaled(torch.autograd.Function):
    """x times the number of the pass and one, which autograd keeps the pass for."""

    @staticmethod
    def forward(ctx, x, one):
        ctx.one = one
        ctx.save_for_backward(x)
        return x * (one.number + 1)

    @staticmethod
    def backward(ctx, dy):
        ctx.saved_tensors
        return dy * (ctx.one.number + 1), None


def step(model, seen):
    def run(x):
        one = model._drop_pass()
        seen.append(one.number)
        return Scaled.apply(x, one).square().sum()   # (the square saves its input: it is computed again)
    return run


def test_every_pass_has_a_number_of_its_own_and_a_recomputed_one_the_same():
    model, seen = model_of(), []
    x = torch.ones(3, requires_grad=True)
    losses = [checkpoint(step(model, seen), x, use_reentrant=False) for _ in range(3)]
    assert seen == [0, 1, 2] and model.drop_passes == 3
    sum(losses).backward()
    assert sorted(seen[3:]) == [0, 1, 2] and model.drop_passes == 3
    assert (x.grad == 2 * (1 + 4 + 9)).all()
    torch.manual_seed(5)   # the same numbers from torch's generator again: still a new pass
    first = step(model, seen)(x)
    torch.manual_seed(5)
    second = step(model, seen)(x)
    assert seen[-2:] == [3, 4] and model.drop_passes == 5
    del losses, first, second
    gc.collect()
    assert len(model._drop_known) == 0   # nothing is held longer than its graph


@pytest.mark.parametrize("how", [dict(use_reentrant=False, preserve_rng_state=False), dict(use_reentrant=True)])
def test_a_recomputed_pass_that_is_not_known_is_refused(how):
    model, seen = model_of(), []
    run = step(model, seen)
    if how["use_reentrant"]:   # (the first run is one without gradients, which drops nothing)
        run = lambda x: step(model, seen)(x) if torch.is_grad_enabled() else x.square().sum()  # noqa: E731
    loss = checkpoint(run, torch.ones(3, requires_grad=True), **how)
    with pytest.raises(RuntimeError, match="use_reentrant=False"):
        loss.backward()


def test_passes_that_began_alike_are_not_taken_for_one_another():
    model, seen = model_of(), []
    x = torch.ones(3, requires_grad=True)
    losses = []
    for _ in range(2):
        torch.manual_seed(7)
        losses.append(checkpoint(step(model, seen), x, use_reentrant=False))
    assert seen == [0, 1]
    for loss in losses:
        with pytest.raises(RuntimeError, match="seeded alike"):
            loss.backward()
    del losses, loss
    gc.collect()
    for k in (2, 3):   # one after the other they are
        torch.manual_seed(7)
        loss = checkpoint(step(model, seen), x, use_reentrant=False)
        loss.backward()
        assert seen[-2:] == [k, k]
        del loss
