"""A small recurrent language model that runs the operators of this package together: embedding, layer norms, Gated Delta
Rule scans (``jit``), a layer norm of each head, log probabilities; as options rotary positions on queries and keys, a gated
feed-forward block behind each scan, and a loss without logits.

    python -m flex_rnn_b200.language_model                  # trains on synthetic text, scores it, continues it
    python -m flex_rnn_b200.language_model --hidden 704 --turned 32 --without-logits

Training: ``model.loss(tokens)`` and its gradients.  Scoring: ``model.score(tokens, top=5)``.  Generation: ``model.generate``
reads a prompt once and then one token a call, with the layers' states handed on.  ``plain=True`` computes the same from
the operators' definitions in plain PyTorch, on any device and in any precision.
"""
from __future__ import annotations

import argparse
from typing import List, Optional, Tuple, Union

import torch
import torch.nn.functional as F
from torch import nn

from . import lm
from .jit import jit
from .workloads import gated_delta_rule

scan = jit(gated_delta_rule)


class Layer(nn.Module):
    """x + W_out norm_of_heads(scan(projections of norm(x) at this place and the one before)).  Its state: the scan's,
    norm(x) of the last place, and the next place's position.  ``turned`` values of each head's query and key carry rotary positions; with ``hidden``, a gated
    feed-forward block of that many values follows: x + block(norm(x))."""

    def __init__(self, width: int, heads: int, head_width: int, hidden: int = 0, turned: int = 0):
        super().__init__()
        self.heads, self.head_width = heads, head_width
        n = heads * head_width
        self.norm_weight, self.norm_bias = nn.Parameter(torch.ones(width)), nn.Parameter(torch.zeros(width))
        self.project = nn.Linear(2 * width, 3 * n + 2 * heads, bias=False)
        self.head_weight, self.head_bias = nn.Parameter(torch.ones(heads, head_width)), nn.Parameter(torch.zeros(heads, head_width))
        self.out = nn.Linear(n, width, bias=False)
        self.hidden, self.turned = hidden, turned
        if turned:
            # (no buffer: a model that changes its type keeps its frequencies in 64 bits; _apply takes them along)
            self.frequencies = lm.rotary_frequencies(turned, base=500.0)
        if hidden:
            self.block_weight, self.block_bias = nn.Parameter(torch.ones(width)), nn.Parameter(torch.zeros(width))
            self.gate, self.up, self.down = nn.Linear(width, hidden, bias=False), nn.Linear(width, hidden, bias=False), nn.Linear(hidden, width, bias=False)

    def _apply(self, fn, *args, **kwargs):
        super()._apply(fn, *args, **kwargs)
        if self.turned:                   # (a copy from the host has no place in a call: that may be captured into a graph)
            self.frequencies = lm.rotary_frequencies(self.turned, base=500.0).to(self.norm_weight.device)
        return self

    def forward(self, x, state, ops, position: Optional[int] = None):
        B, T, _ = x.shape
        H, M = self.heads, self.head_width
        state, last, *at = state          # (without a position: at the beginning)
        if position is None:
            position = at[0] if at else 0
        h = ops.layer_norm(x, self.norm_weight, self.norm_bias)
        before = torch.cat([last[:, None], h[:, :-1]], 1)
        q, k, v, g, beta = self.project(torch.cat([h, before], -1)).split([H * M, H * M, H * M, H, H], dim=-1)
        # (padding has zero vectors; 1e-12, the usual bound, is zero in fp16)
        row = lambda t: F.normalize(t.view(B, T, H, 1, M), dim=-1, eps=max(1e-12, torch.finfo(t.dtype).tiny))
        scalar = lambda t: torch.sigmoid(t).view(B, T, H, 1, 1)
        q, k = row(q), row(k)
        if self.turned:
            f = self.frequencies.to(x.device)      # (there already, unless parameters were replaced one by one)
            q, k = ops.rotary(q, position, f), ops.rotary(k, position, f)
        # states are kept in 32 bits from call to call; the outputs have their type
        y, state = ops.scan(q, k, v.reshape(B, T, H, M, 1), scalar(g + 3), scalar(beta), state)
        y = ops.layer_norm(y.to(x.dtype), self.head_weight, self.head_bias)
        x = x + self.out(y.reshape(B, T, H * M))
        if self.hidden:
            x = x + ops.gated_mlp(ops.layer_norm(x, self.block_weight, self.block_bias), self.gate.weight, self.up.weight, self.down.weight)
        return x, (state, h[:, -1], position + T)


class _Fast:
    embedding, layer_norm, token_logprobs, scan = staticmethod(lm.embedding), staticmethod(lm.layer_norm), staticmethod(lm.token_logprobs), staticmethod(scan)
    rotary, gated_mlp, linear_logprobs = staticmethod(lm.rotary), staticmethod(lm.gated_mlp), staticmethod(lm.linear_logprobs)


class _Plain:
    embedding, layer_norm, token_logprobs = staticmethod(lm.naive_embedding), staticmethod(lm.naive_layer_norm), staticmethod(lm.naive_token_logprobs)
    rotary, gated_mlp, linear_logprobs = staticmethod(lm.naive_rotary), staticmethod(lm.naive_gated_mlp), staticmethod(lm.naive_linear_logprobs)

    @staticmethod
    def scan(*args):
        return scan.naive(*args, dtype=args[-1].dtype)


class RecurrentLM(nn.Module):
    """``hidden`` and ``turned``: see ``Layer``.  Without ``keep_logits``, ``loss`` and scores without alternatives are computed
    from the vectors before the last projection."""

    def __init__(self, vocabulary: int, width: int = 256, layers: int = 2, heads: int = 4, head_width: int = 64, plain: bool = False, hidden: int = 0, turned: int = 0, keep_logits: bool = True):
        super().__init__()
        self.keep_logits = keep_logits
        self.ops = _Plain if plain else _Fast
        self.scale = width ** 0.5
        self.weight = nn.Parameter(torch.randn(vocabulary, width) * width ** -0.5)
        self.layers = nn.ModuleList(Layer(width, heads, head_width, hidden, turned) for _ in range(layers))
        self.norm_weight, self.norm_bias = nn.Parameter(torch.ones(width)), nn.Parameter(torch.zeros(width))
        self.head = nn.Linear(width, vocabulary, bias=False)

    def states(self, batch: int) -> List[Tuple[torch.Tensor, torch.Tensor, int]]:
        p = self.weight
        dtype = torch.promote_types(p.dtype, torch.float32)
        return [(torch.zeros(batch, l.heads, l.head_width, l.head_width, dtype=dtype, device=p.device), p.new_zeros(batch, p.shape[1]), 0) for l in self.layers]

    def features(self, tokens, states: Optional[list] = None, position: Optional[int] = None) -> Tuple[torch.Tensor, list]:
        """tokens [B,T] (``-100``: padding, a zero input), the layers' states, the first token's position (default: the one after
        those that the states have seen) -> what the last projection takes [B,T,width], new states"""
        states = self.states(tokens.shape[0]) if states is None else states
        x, new = self.ops.embedding(tokens, self.weight, scale=self.scale), []
        for layer, state in zip(self.layers, states):
            x, state = layer(x, state, self.ops, position)
            new.append(state)
        return self.ops.layer_norm(x, self.norm_weight, self.norm_bias), new

    def forward(self, tokens, states: Optional[list] = None, position: Optional[int] = None) -> Tuple[torch.Tensor, list]:
        """As ``features``, but with logits [B,T,vocabulary]."""
        x, new = self.features(tokens, states, position)
        return self.head(x), new

    def score(self, tokens, top: int = 0, temperature: float = 1.0) -> Union[lm.TokenLogprobs, lm.LinearLogprobs]:
        """Log probability of each token but the first of tokens [B,T] after those before it; padding counts as 0."""
        if not self.keep_logits and not top:
            return self.ops.linear_logprobs(self.features(tokens[:, :-1])[0], self.head.weight, tokens[:, 1:], temperature=temperature)
        logits, _ = self(tokens[:, :-1])
        return self.ops.token_logprobs(logits, tokens[:, 1:], top=top, temperature=temperature)

    def loss(self, tokens, entropy_weight: float = 0.0) -> torch.Tensor:
        """Mean negative log probability of the tokens that are no padding, less a bonus for entropy."""
        r = self.score(tokens)
        there = tokens[:, 1:] != -100
        return -(r.logprob + entropy_weight * torch.where(there, r.entropy, 0.0)).sum() / there.sum()

    @torch.no_grad()
    def generate(self, prompt, steps: int, temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
        """The most probable continuation, token by token, of prompt [B,T]: tokens [B,steps] and their log probabilities."""
        logits, states = self(prompt)
        last, tokens, logprobs = logits[:, -1], [], []
        for _ in range(steps):
            # (the alternatives come with the log probability of any token; 0 stands in for it)
            best = self.ops.token_logprobs(last, torch.zeros_like(prompt[:, 0]), top=1, temperature=temperature)
            tokens.append(best.top_token)
            logprobs.append(best.top_logprob)
            logits, states = self(best.top_token, states)
            last = logits[:, 0]
        return torch.cat(tokens, 1), torch.cat(logprobs, 1)


def synthetic_text(batch: int, length: int, vocabulary: int, seed: int = 0) -> torch.Tensor:
    """Sequences that repeat a random phrase of eight tokens, with padding behind some of them."""
    g = torch.Generator().manual_seed(seed)
    phrase = torch.randint(0, vocabulary, (batch, 8), generator=g)
    text = phrase.repeat(1, -(-length // 8))[:, :length].contiguous()
    ends = torch.randint(length // 2, length + 1, (batch, 1), generator=g)
    return torch.where(torch.arange(length) < ends, text, -100)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--length", type=int, default=128)
    ap.add_argument("--vocabulary", type=int, default=512)
    ap.add_argument("--hidden", type=int, default=0, help="values of a gated feed-forward block behind each scan (0: none)")
    ap.add_argument("--turned", type=int, default=0, help="values of each head's query and key that carry rotary positions")
    ap.add_argument("--without-logits", action="store_true", help="the loss from the vectors before the last projection")
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    model = RecurrentLM(a.vocabulary, hidden=a.hidden, turned=a.turned, keep_logits=not a.without_logits).cuda()
    optimiser = torch.optim.AdamW(model.parameters(), lr=3e-3)
    for step in range(a.steps):
        loss = model.loss(synthetic_text(a.batch, a.length, a.vocabulary, seed=step).cuda(), entropy_weight=0.001)
        optimiser.zero_grad(set_to_none=True)
        loss.backward()
        optimiser.step()
        if step % 20 == 0 or step == a.steps - 1:
            print(f"step {step}: loss {float(loss.detach()):.3f}")
    text = synthetic_text(2, 64, a.vocabulary, seed=a.steps).clamp_min(0).cuda()
    with torch.no_grad():
        r = model.score(text, top=3)
    print("log probability of the last eight tokens of a new text:", [f"{v:.2f}" for v in r.logprob[0, -8:].tolist()])
    tokens, logprobs = model.generate(text[:, :32], 8)
    print("its continuation:", tokens[0].tolist(), "its phrase:", text[0, 32:40].tolist())


if __name__ == "__main__":
    main()
