"""The operators together, as the small recurrent language model runs them."""
import copy

import pytest
import torch

from flex_rnn_b200.language_model import RecurrentLM, synthetic_text


def make(dtype, plain, device):
    torch.manual_seed(1)
    return RecurrentLM(97, width=48, layers=2, heads=3, head_width=16, plain=plain).to(device, dtype)


def test_plain_model_on_the_cpu():
    """Definitions alone: one pass equals token by token, padding changes nothing before it, gradients arrive everywhere."""
    model = make(torch.float64, True, "cpu")
    text = synthetic_text(3, 20, 97)
    whole, _ = model(text)
    states, parts = None, []
    for t in range(20):
        logits, states = model(text[:, t:t + 1], states)
        parts.append(logits)
    assert torch.allclose(whole, torch.cat(parts, 1), atol=1e-10)
    loss = model.loss(text, entropy_weight=0.1)
    loss.backward()
    assert loss.isfinite() and all(p.grad is not None and p.grad.isfinite().all() and p.grad.any() for p in model.parameters())


@pytest.mark.gpu
def test_model_equals_its_plain_form():
    """Loss, scores and gradients in fp32 against 64 bits: about ten operators in a row, each with a relative error of a few
    2^-24 and a condition of some tens (norms of rows of 16 to 48)."""
    fast, plain = make(torch.float32, False, "cuda"), make(torch.float64, True, "cuda")
    plain.load_state_dict({k: v.double() for k, v in fast.state_dict().items()})
    text = synthetic_text(3, 24, 97).cuda()
    a, b = fast.loss(text, entropy_weight=0.1), plain.loss(text, entropy_weight=0.1)
    assert abs(float(a.detach()) - float(b.detach())) <= 1e-5 * abs(float(b.detach()))
    a.backward()
    b.backward()
    for (name, p), q in zip(fast.named_parameters(), plain.parameters()):
        assert float((p.grad.double() - q.grad).norm()) <= 2e-4 * float(q.grad.norm()) + 1e-9, name
    with torch.no_grad():
        r, s = fast.score(text, top=4), plain.score(text, top=4)
    assert float((r.logprob.double() - s.logprob).abs().max()) <= 1e-3 and float((r.entropy.double() - s.entropy).abs().max()) <= 1e-3
    assert float((r.top_logprob.double() - s.top_logprob).abs().max()) <= 1e-3


@pytest.mark.gpu
def test_training_and_generation():
    """The loss of repeated phrases falls; a prompt read at once and token by token give the same continuation."""
    torch.manual_seed(0)
    model = RecurrentLM(64, width=128, layers=2, heads=2, head_width=64).cuda()
    optimiser = torch.optim.AdamW(model.parameters(), lr=3e-3)
    losses = []
    for step in range(60):
        loss = model.loss(synthetic_text(16, 96, 64, seed=step).cuda())
        optimiser.zero_grad(set_to_none=True)
        loss.backward()
        optimiser.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < 0.75 * losses[0]
    prompt = synthetic_text(2, 32, 64, seed=999).clamp_min(0).cuda()
    tokens, logprobs = model.generate(prompt, 6)
    with torch.no_grad():
        r = model.score(torch.cat([prompt, tokens], 1), top=1)
    assert torch.equal(r.top_token[:, -6:, 0], tokens)
    assert torch.allclose(r.logprob[:, -6:], logprobs, atol=1e-3)


@pytest.mark.gpu
def test_half_precision_model():
    """bf16 weights and activations: the loss agrees with the fp32 model's to bf16's rounding over the layers."""
    full = make(torch.float32, False, "cuda")
    half = copy.deepcopy(full).bfloat16()
    text = synthetic_text(4, 40, 97).cuda()
    a, b = full.loss(text), half.loss(text)
    b.backward()
    assert abs(float(a.detach()) - float(b.detach())) <= 0.05 * float(a.detach())
    assert all(p.grad.isfinite().all() and p.grad.dtype == torch.bfloat16 for p in half.parameters())
