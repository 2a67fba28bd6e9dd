"""A decoder with a gated layer, rotary positions and dropout whose QKV weights are in tables of their own, as several ranks have them
(on one rank, which has all rows)."""
import pytest
import torch
from test_gpt_fused_autograd_gpu import close, grads, once
from test_gpt_gated_gpu import SIZES, batch

from parameter_server_b200.models.gpt import GPT, GPTConfig
from parameter_server_b200.ops.dense import DenseTable

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 8])
def test_qkv_weights_in_tables_of_their_own(bits):
    model = GPT(GPTConfig(**SIZES, gated=True, rotary=True, dropout=0.1, act_bits=bits), seed=1)
    loss0, one = once(model)
    d = SIZES["d_model"]
    for i in range(SIZES["n_layer"]):
        table = DenseTable({"w": (3 * d, d)}, "adamw", dict(lr=SIZES["lr"]), grad_dtype=torch.float32, device=model.device, scatter_peers=False)
        table.load({"w": model.main.params[f"h{i}.qkv.w"].detach().float().cpu()})
        table.zero_grads()
        model.qkv[i] = table
    model.zero_grads()
    model.drop_passes = 0   # the same masks again
    _, loss = model.forward(*batch())
    loss.backward()
    two = grads(model)
    for i in range(SIZES["n_layer"]):
        assert (two[f"h{i}.qkv.w"] == 0).all()
        two[f"h{i}.qkv.w"] = model.qkv[i].grads["w"].clone()
    close(two, one)
    assert abs(loss.item() - loss0) < 2e-3   # the product itself is another kernel's
    model.check()
