"""A captured pass of a decoder with dropout draws anew at every replay, and its gradients are those of its own masks."""
import pytest
import torch
from test_gpt_gated_gpu import SIZES, batch, reference

from parameter_server_b200.models.gpt import GPT, GPTConfig

pytestmark = pytest.mark.gpu


def captured(model, tokens, targets):
    """A graph of a pass and its backward pass; the loss, and the gradients of the leaves."""
    def run():
        loss = model.forward(tokens, targets)[1]
        loss.backward()
        return loss.detach(), {n: p.grad for n, p in model._leaves.items()}

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):   # once outside, as a capture wants it; nothing of its graph lives on
        run()
    torch.cuda.current_stream().wait_stream(side)
    model.zero_grads()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    return graph, *out


@pytest.mark.parametrize("parts", [dict(dropout=0.2), dict(gated=True, rotary=True, dropout=0.1)])
def test_every_replay_draws_anew(parts):
    model = GPT(GPTConfig(**SIZES, **parts), seed=1)
    tokens, targets = batch()

    graph, loss, leaves = captured(model, tokens, targets)
    assert model.drop_passes == 2
    base, losses = model.drop_seed, []
    for replay in (1, 2):
        for t in model.tables:
            t.zero_grads()
        graph.replay()
        torch.cuda.synchronize()
        got = {n: g + leaves[n].float() if n in leaves else g.clone() for n, g in model.main.grads.items()}
        losses.append(loss.item())
        model.drop_seed = base + (replay << 40)   # the seed that a replay draws from
        want, wanted = reference(model, tokens, targets, 1)
        model.drop_seed = base
        assert abs(losses[-1] - want) < 1e-2
        for n in got:
            assert (got[n] - wanted[n]).norm() / wanted[n].norm().clamp_min(1e-12) < 0.05, n
    assert losses[0] != losses[1]
    model.check()


def test_two_passes_of_a_graph_draw_different_masks():
    model = GPT(GPTConfig(**SIZES, dropout=0.5), seed=2)
    tokens, targets = batch()
    graph = torch.cuda.CUDAGraph()
    model.forward(tokens, targets)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        losses = [model.forward(tokens, targets)[1].detach() for _ in range(2)]
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        seen += [v.item() for v in losses]
    assert len(set(seen)) == 6
