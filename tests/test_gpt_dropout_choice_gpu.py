"""Whether a pass of the decoder drops values is the caller's choice, whatever else the call has."""
import pytest
import torch
import torch.nn.functional as F
from test_gpt_gated_gpu import SIZES, batch, reference

from parameter_server_b200.models.gpt import GPT, GPTConfig

pytestmark = pytest.mark.gpu


def test_a_loss_of_ones_own_trains_with_dropout():
    model = GPT(GPTConfig(**SIZES, dropout=0.2), seed=1)
    tokens, targets = batch()
    model.zero_grads()
    logits, none = model.forward(tokens, drop=True)
    assert none is None and model.drop_passes == 1
    loss = F.cross_entropy(logits.float().view(-1, 512), targets.reshape(-1))
    loss.backward()
    torch.cuda.synchronize()
    want, wanted = reference(model, tokens, targets, 0)
    assert abs(loss.item() - want) < 1e-2
    for name in ("h0.fc.w", "h1.proj.w", "h1.ln2.g"):
        assert (model.main.grads[name] - wanted[name]).norm() / wanted[name].norm() < 0.05, name


def test_a_validation_loss_with_gradients_on_may_drop_nothing():
    model, same = (GPT(GPTConfig(**SIZES, dropout=p), seed=3) for p in (0.5, 0.0))
    tokens, targets = batch()
    assert torch.equal(model.forward(tokens, targets, drop=False)[1], same.forward(tokens, targets)[1]) and model.drop_passes == 0
    with torch.no_grad():
        some = [model.forward(tokens, targets, drop=True)[1].item() for _ in range(2)]
    assert model.drop_passes == 2 and some[0] != some[1]
    assert torch.equal(same.forward(tokens, targets, drop=True)[1], same.forward(tokens, targets)[1])   # a model without dropout
