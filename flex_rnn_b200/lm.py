"""Operators that a language model needs around its scans: ``embedding`` before them, ``layer_norm`` before a projection
or over each head of a scan's output, ``token_logprobs`` at the end (loss, scoring, alternatives).

They work on CUDA tensors, on the current stream, forward and backward, in fp32, bf16 or fp16 with arithmetic in 32 bits;
each is one operator for autograd, ``torch.compile`` and CUDA graphs, with hand-written kernels behind it
(csrc/frnn_embedding.cu, frnn_layer_norm.cu, frnn_logprobs.cu).  ``naive_*`` are their definitions in plain PyTorch, for
any device and data type.  Nothing of this is in the reference, which ends at the recurrence.
"""
from __future__ import annotations

import threading
from typing import NamedTuple, Optional

import torch as th

#: The most alternatives that ``token_logprobs`` returns for a row (FRNN_MAX_TOP of include/frnn.h).
MAX_TOP = 32

_ops = th.ops.flex_rnn_b200
_loaded = False
_lock = threading.Lock()


# (under torch.compile this runs while a call is traced and counts as a constant: the first use of an operator may be a
# compiled one, and a tracer can neither enter the lock nor load a library)
@th.compiler.assume_constant_result
def _operators():
    """Load the operators of the native host library, once."""
    global _loaded
    if not _loaded:
        from . import runtime
        with _lock:
            if not _loaded:
                runtime.host()
                _register_fakes()
                _loaded = True


class TokenLogprobs(NamedTuple):
    logprob: th.Tensor          #: fp32, of the shape of the tokens
    entropy: th.Tensor          #: fp32, of the shape of the tokens
    top_logprob: th.Tensor      #: fp32 [..., top]; carries no gradient
    top_token: th.Tensor        #: int64 [..., top]


def embedding(tokens: th.Tensor, weight: th.Tensor, scale: float = 1.0, ignore_index: int = -100) -> th.Tensor:
    """``scale * weight[tokens]``: ``[*tokens.shape, width]`` of the type of ``weight`` [vocabulary, width].

    ``tokens`` are int64 or int32.  Places with ``ignore_index`` give zeros and add to no gradient.  A token outside the
    vocabulary gives zeros too and is reported: the next call on that GPU raises ``FrnnError`` (no call waits for the GPU
    to look).  The gradient of ``weight`` is dense and sums each token's rows in 32 bits, in an order that the
    tokens' places, the sizes and the GPU's number of SMs fix, so it is the same in every run."""
    _operators()
    return _ops.embedding.default(tokens, weight, scale, ignore_index)


def layer_norm(x: th.Tensor, weight: Optional[th.Tensor] = None, bias: Optional[th.Tensor] = None, eps: float = 1e-5) -> th.Tensor:
    """``(x - mean) / sqrt(variance + eps) * weight + bias`` over the last dimension of ``x``.

    ``weight`` and ``bias`` are [width], or [heads, width] for ``x`` [..., heads, width] (a norm of each head, as on the
    output [B,T,H,M] of a scan), of the type of ``x`` or fp32.  ``x`` may have any strides; layouts whose rows are not
    runs of consecutive elements, or that need more than three strides between rows, are copied first."""
    _operators()
    return _ops.layer_norm.default(x, weight, bias, eps, False)[0]


def token_logprobs(logits: th.Tensor, tokens: th.Tensor, top: int = 0, temperature: float = 1.0, ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of ``tokens`` [...] under ``softmax(logits / temperature)``, ``logits`` [..., vocabulary], the
    entropy of each row, and its ``top`` largest alternatives (at most ``MAX_TOP``; equal logits: the lowest token first).

    Logits may be -inf (tokens that a mask forbids): they have probability 0 and add nothing to the entropy.  A row that
    is -inf throughout has log probabilities -inf, entropy 0 and gradient 0.  Tokens equal to ``ignore_index`` have log
    probability 0 and no gradient through it; tokens outside the vocabulary have NaN, and the next call on that GPU raises
    ``FrnnError``.  ``logprob`` and ``entropy`` are differentiable; the alternatives carry no gradient.  A NaN logit, or
    +inf, makes its row's results NaN."""
    _operators()
    return TokenLogprobs(*_ops.token_logprobs.default(logits, tokens, top, temperature, ignore_index, False)[:4])


# ---- definitions ---------------------------------------------------------------------------------------------------------

def naive_embedding(tokens, weight, scale=1.0, ignore_index=-100):
    """Definition of ``embedding`` in the arithmetic of ``weight``; tokens outside the vocabulary are errors."""
    there = tokens != ignore_index
    return weight[th.where(there, tokens, 0)] * scale * there.unsqueeze(-1)


def naive_layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Definition of ``layer_norm`` in the arithmetic of ``x``."""
    c = x - x.mean(-1, True)
    y = c * (c.square().mean(-1, True) + eps).rsqrt()
    y = y if weight is None else y * weight
    return y if bias is None else y + bias


def naive_token_logprobs(logits, tokens, top=0, temperature=1.0, ignore_index=-100):
    """Definition of ``token_logprobs`` in the arithmetic of ``logits``."""
    none = (logits == -th.inf).all(-1, True)
    logp = th.log_softmax(th.where(none, 0.0, logits) / temperature, -1)
    p = logp.exp()
    entropy = -th.where(none | (p == 0), 0.0, p * th.where(p == 0, 0.0, logp)).sum(-1)
    logp = th.where(none, -th.inf, logp)
    there = tokens != ignore_index
    lp = th.where(there, logp.gather(-1, th.where(there, tokens, 0).unsqueeze(-1)).squeeze(-1), 0.0)
    best = th.sort(logits.detach(), dim=-1, descending=True, stable=True).indices[..., :top]
    return TokenLogprobs(lp, entropy, logp.detach().gather(-1, best), best)


# ---- shapes for torch.compile ----------------------------------------------------------------------------------------------

def _register_fakes():
    fake = th.library.register_fake

    @fake("flex_rnn_b200::embedding")
    def _(tokens, weight, scale, ignore_index):
        return weight.new_empty((*tokens.shape, weight.shape[1]))

    @fake("flex_rnn_b200::embedding_backward")
    def _(grad, tokens, rows, scale, ignore_index):
        return grad.new_empty((rows, grad.shape[-1]))

    @fake("flex_rnn_b200::layer_norm")
    def _(x, weight, bias, eps, save):
        rows = x.numel() // x.shape[-1] if save and x.shape[-1] else 0
        return x.new_empty(x.shape), x.new_empty((rows, 2), dtype=th.float32)

    @fake("flex_rnn_b200::layer_norm_backward")
    def _(grad, x, weight, bias, stats, want_x, want_weight, want_bias):
        none = x.new_empty((0,))
        like = lambda p, want: p.new_empty(p.shape) if want and p is not None else none.clone()
        return th.empty_like(x) if want_x else none, like(weight, want_weight), like(bias, want_bias)

    @fake("flex_rnn_b200::token_logprobs")
    def _(logits, tokens, top, temperature, ignore_index, save):
        new = lambda *shape, dtype=th.float32: logits.new_empty(shape, dtype=dtype)
        s = tokens.shape
        return new(*s), new(*s), new(*s, top), new(*s, top, dtype=th.int64), new(tokens.numel() if save else 0, 3)

    @fake("flex_rnn_b200::token_logprobs_backward")
    def _(dlogprob, dentropy, logits, tokens, stats, temperature, ignore_index):
        return logits.new_empty(logits.shape)
