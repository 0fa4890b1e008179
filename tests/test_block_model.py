"""The language model with its feed-forward blocks, rotary positions and its loss without logits: the operators in a run."""
import copy

import pytest
import torch

from flex_rnn_b200.language_model import RecurrentLM, main, synthetic_text

PARTS = dict(hidden=80, turned=12, keep_logits=False)


def make(dtype, plain, device, **parts):
    torch.manual_seed(1)
    return RecurrentLM(97, width=48, layers=2, heads=3, head_width=16, plain=plain, **{**PARTS, **parts}).to(device, dtype)


def test_plain_model_on_the_cpu():
    """Definitions alone: one pass equals token by token with positions that go on, the loss is that from logits, and gradients
    arrive everywhere."""
    model = make(torch.float64, True, "cpu")
    text = synthetic_text(3, 20, 97)
    whole, _ = model(text)
    states, parts = None, []
    for t in range(20):
        logits, states = model(text[:, t:t + 1], states, t)
        parts.append(logits)
    assert torch.allclose(whole, torch.cat(parts, 1), atol=1e-10)
    other = make(torch.float64, True, "cpu", keep_logits=True)
    loss = model.loss(text, entropy_weight=0.1)
    assert torch.allclose(loss, other.loss(text, entropy_weight=0.1), rtol=1e-12)
    loss.backward()
    assert loss.isfinite() and all(p.grad is not None and p.grad.isfinite().all() and p.grad.any() for p in model.parameters())


def test_default_model_is_what_it_was():
    """Without the options there are no further parameters, drawn in no other order."""
    torch.manual_seed(1)
    names = [n for n, _ in RecurrentLM(97, width=48, layers=1, heads=3, head_width=16).named_parameters()]
    assert names == ["weight", "norm_weight", "norm_bias", "layers.0.norm_weight", "layers.0.norm_bias", "layers.0.head_weight", "layers.0.head_bias", "layers.0.project.weight", "layers.0.out.weight",
                     "head.weight"]


@pytest.mark.gpu
def test_model_equals_its_plain_form():
    """Loss, scores and gradients in fp32 against 64 bits: some fifteen operators in a row, each with a relative error of a few
    2^-24 (products on the tensor cores a few 2^-21) and a condition of some tens (norms of rows of 16 to 48)."""
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
        r, s = fast.score(text), plain.score(text)
        assert float((r.logprob.double() - s.logprob).abs().max()) <= 1e-3 and float((r.entropy.double() - s.entropy).abs().max()) <= 1e-3
        top = fast.score(text, top=3)
        assert float((top.logprob - r.logprob).abs().max()) <= 1e-3 and top.top_token.shape == (3, 23, 3)


@pytest.mark.gpu
def test_generation_token_by_token():
    """A prompt read at once and token by token give the same continuation, with positions that go on."""
    torch.manual_seed(0)
    model = RecurrentLM(64, width=128, layers=2, heads=2, head_width=64, hidden=200, turned=64, keep_logits=False).cuda()
    prompt = synthetic_text(2, 32, 64, seed=999).clamp_min(0).cuda()
    tokens, logprobs = model.generate(prompt, 6)
    with torch.no_grad():
        r = model.score(torch.cat([prompt, tokens], 1), top=1)
        q = model.score(torch.cat([prompt, tokens], 1))
    assert torch.equal(r.top_token[:, -6:, 0], tokens)
    assert torch.allclose(r.logprob[:, -6:], logprobs, atol=1e-3) and torch.allclose(q.logprob, r.logprob, atol=1e-3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_half_precision_model(dtype):
    """16-bit weights and activations: the loss agrees with the fp32 model's to that rounding over the layers."""
    full = make(torch.float32, False, "cuda")
    half = copy.deepcopy(full).to(dtype)
    text = synthetic_text(4, 40, 97).cuda()
    a, b = full.loss(text), half.loss(text)
    b.backward()
    assert abs(float(a.detach()) - float(b.detach())) <= 0.05 * float(a.detach())
    assert all(p.grad.isfinite().all() and p.grad.dtype == dtype for p in half.parameters())


@pytest.mark.gpu
def test_training_step_in_a_graph():
    """A whole training pass captured and replayed gives what it gives eagerly."""
    model = make(torch.bfloat16, False, "cuda")
    text = synthetic_text(4, 33, 97).clamp_min(0).cuda()
    params = list(model.parameters())

    def step():
        loss = model.loss(text, entropy_weight=0.1)
        return [loss.detach(), *torch.autograd.grad(loss, params)]

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_command(capsys):
    main(["--steps", "2", "--batch", "2", "--length", "24", "--vocabulary", "64", "--hidden", "40", "--turned", "8", "--without-logits"])
    assert "continuation" in capsys.readouterr().out
