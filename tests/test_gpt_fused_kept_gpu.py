"""What a fused decoder holds between its forward and its backward pass."""
import pytest
import torch

from parameter_server_b200.models.gpt import GPT, GPTConfig

pytestmark = pytest.mark.gpu

D, HEADS, HIDDEN, SEQ, BATCH = 512, 8, 2048, 1024, 4


def tokens():
    return torch.randint(0, 512, (BATCH, SEQ), generator=torch.Generator().manual_seed(0)).cuda()


def requested():
    torch.cuda.synchronize()
    return torch.cuda.memory_stats()["requested_bytes.all.current"]


def held(layers, bits):
    """Bytes that a forward pass leaves behind."""
    model = GPT(GPTConfig(n_layer=layers, d_model=D, n_head=HEADS, d_ff=HIDDEN, vocab=512, seq_len=SEQ, fused=True, act_bits=bits), seed=1)
    t = tokens()
    _, loss = model.forward(t, t)
    loss.backward()   # (whatever is made once is there)
    del loss
    before = requested()
    _, loss = model.forward(t, t)
    return requested() - before


@pytest.mark.parametrize("bits", [16, 8])
def test_a_layer_keeps_what_its_backward_pass_needs_once(bits):
    """Per token: q, k, v and attention's output in 16 bits with a sum per head, and of two norms and the hidden layer either 8 bits, a
    byte per 32 of them and a root, or 16 bits: the norms' inputs and outputs with mean and root, and the hidden layer."""
    attention = 2 * 4 * D + 4 * HEADS
    if bits == 8:
        rest = 2 * (D + D // 32 + 4) + HIDDEN + HIDDEN // 32
    else:
        rest = 2 * (2 * 2 * D + 8) + 2 * HIDDEN
    per_token = (held(4, bits) - held(2, bits)) / 2 / (BATCH * SEQ)
    assert per_token <= 1.02 * (attention + rest), (per_token, attention + rest)


def peak(layers, bits):
    """Bytes above what was there that a forward pass asks for at most, where no backward pass can follow; and its result."""
    model = GPT(GPTConfig(n_layer=layers, d_model=D, n_head=HEADS, d_ff=HIDDEN, vocab=512, seq_len=SEQ, fused=True, act_bits=bits), seed=1)
    t = tokens()
    with torch.no_grad():
        model.forward(t)
        before = requested()
        torch.cuda.reset_peak_memory_stats()
        logits, _ = model.forward(t)
        torch.cuda.synchronize()
    return torch.cuda.memory_stats()["requested_bytes.all.peak"] - before, logits, model.forward(t)[0].detach()


@pytest.mark.parametrize("bits", [16, 8])
def test_a_forward_pass_alone_makes_no_checkpoints(bits):
    """The most is held where the hidden layer is there beside x, the norm's output and the block's, whatever the model would keep of
    them; and the values are those of a training pass."""
    top, logits, training = peak(2, bits)
    assert torch.equal(logits, training)
    n = BATCH * SEQ
    assert top <= 1.02 * n * (2 * HIDDEN + 3 * 2 * D + 8) + (1 << 20), (top / n, 2 * HIDDEN + 3 * 2 * D + 8)
    assert peak(4, bits)[0] <= 1.001 * top


def test_inference_mode_runs_a_fused_model():
    t = tokens()
    for bits in (16, 8):
        model = GPT(GPTConfig(n_layer=2, d_model=D, n_head=HEADS, d_ff=HIDDEN, vocab=512, seq_len=SEQ, fused=True, act_bits=bits), seed=1)
        want = model.forward(t)[0].detach()
        with torch.inference_mode():
            assert torch.equal(model.forward(t)[0], want)
