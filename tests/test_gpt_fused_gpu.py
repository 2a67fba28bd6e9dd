"""The decoder on the block operators against the same decoder on torch ops: loss, gradients, optimizer steps."""
import pytest
import torch

from parameter_server_b200.models.gpt import GPT, GPTConfig

pytestmark = pytest.mark.gpu

SIZES = dict(n_layer=2, d_model=256, n_head=4, d_ff=1024, vocab=512, seq_len=64, lr=3e-3, weight_decay=0.0)


def models(bits):
    """Two models with the same parameters: on torch ops, and fused."""
    return GPT(GPTConfig(**SIZES), seed=1), GPT(GPTConfig(**SIZES, fused=True, act_bits=bits), seed=1)


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


# A bf16 model's gradients carry one rounding of 2^-9 per tensor on the way back, about ten of them deep here: both sides are
# within a few percent of the true gradient in norm. 8-bit checkpoints add about 1 % of a block's values per checkpoint.
@pytest.mark.parametrize("bits,limit", [(16, 0.05), (8, 0.08)])
def test_loss_and_gradients_match_the_model_on_torch_ops(bits, limit):
    plain, fused = models(bits)
    tokens, targets = batch()
    l0, g0 = grads_of(plain, tokens, targets)
    l1, g1 = grads_of(fused, tokens, targets)
    fused.check()
    assert abs(l0 - l1) < 1e-2
    for name in g0:
        off = (g1[name] - g0[name]).norm() / g0[name].norm().clamp_min(1e-12)
        assert off < limit, (name, off.item())


@pytest.mark.parametrize("bits", [16, 8])
def test_training_reduces_the_loss(bits):
    _, model = models(bits)
    tokens, targets = batch()
    losses = [model.train_step(tokens, targets, micro_batches=2).item() for _ in range(12)]
    model.check()
    assert losses[-1] < losses[0] - 0.5, losses


def test_fewer_bits_need_the_fused_blocks():
    with pytest.raises(ValueError, match="act_bits"):
        GPT(GPTConfig(**SIZES, act_bits=8))
    with pytest.raises(ValueError, match="act_bits"):
        GPT(GPTConfig(**SIZES, fused=True, act_bits=4))
