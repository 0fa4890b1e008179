"""Operators that a language model needs around its scans: ``embedding`` before them, ``layer_norm`` before a projection
or over each head of a scan's output, ``rotary`` positions on queries and keys, ``gated_mlp`` between scans, and at the end
``token_logprobs`` (loss, scoring, alternatives from logits) or ``linear_logprobs`` (loss and scoring from the vectors before
the last projection, without logits).

They work on CUDA tensors, on the current stream, forward and backward, in fp32, bf16 or fp16 with arithmetic in 32 bits;
each is one operator for autograd, ``torch.compile`` and CUDA graphs, with hand-written kernels behind it
(csrc/frnn_embedding.cu, frnn_layer_norm.cu, frnn_logprobs.cu, frnn_gated_mlp.cu, frnn_linear_logprobs.cu, frnn_rotary.cu).
``naive_*`` are their definitions in plain PyTorch, for
any device and data type.  Nothing of this is in the reference, which ends at the recurrence.
"""
from __future__ import annotations

import math
import threading
from typing import NamedTuple, Optional, Union

import torch as th

#: The most alternatives that ``token_logprobs`` returns for a row (FRNN_MAX_TOP of include/frnn.h).
MAX_TOP = 32

#: The activations of ``gated_mlp``, in the order of FRNN_SILU ... of include/frnn.h (gelu: the exact one, with erf).
ACTIVATIONS = ("silu", "gelu", "relu", "sigmoid")

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


class LinearLogprobs(NamedTuple):
    logprob: th.Tensor          #: fp32, of the shape of the tokens
    entropy: th.Tensor          #: fp32, of the shape of the tokens


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


def linear_logprobs(x: th.Tensor, weight: th.Tensor, tokens: th.Tensor, temperature: float = 1.0, ignore_index: int = -100) -> LinearLogprobs:
    """``token_logprobs(x @ weight.T, tokens, ...)`` without the logits: log probabilities of ``tokens`` [...] and entropies
    from the vectors ``x`` [..., width] and the last projection's ``weight`` [vocabulary, width], of one type.

    The products run on the tensor cores, with sums in 32 bits (of fp32 as in ``gated_mlp``); the logits leave them a tile at a time and are not kept
    (the forward's workspace holds 12 bytes for each row and 64 or 128 of them, of as many rows at once as 256 MB have room for, but 256), and
    the backward computes them again, a piece of the vocabulary at a time (its workspace holds 2^28 of their gradients, in
    fp32 2^27, or 256 columns where there are more rows).  In bf16 and fp16 their gradient is rounded to that type before it
    is multiplied with ``weight`` and ``x`` (up to 128 rows, ignored ones among them, to twice its bits).  In fp16 a power of two, one for the call, brings
    the largest upstream gradient into range: values of the logits' gradient 2^27 times smaller than that lose bits, below 2^-37 of it they are zero,
    so that a single row of very large gradients takes them from the others.  (Ignored tokens' gradients and rows that are not finite do not count.)
    Results are fp32 and both differentiable.  Tokens equal to ``ignore_index`` have log probability 0 and no gradient through it; tokens outside the
    vocabulary have NaN, and the next call on that GPU raises ``FrnnError``."""
    _operators()
    return LinearLogprobs(*_ops.linear_logprobs.default(x, weight, tokens, temperature, ignore_index, False)[:2])


def gated_mlp(x: th.Tensor, gate: th.Tensor, up: th.Tensor, down: th.Tensor, activation: str = "silu") -> th.Tensor:
    """The gated feed-forward block ``(act(x @ gate.T) * (x @ up.T)) @ down.T``: ``x`` [..., width], ``gate`` and ``up``
    [hidden, width], ``down`` [out, hidden] (as ``nn.Linear`` keeps its weights), all of one type; ``activation`` is one of
    ``ACTIVATIONS``.

    The products run on the tensor cores, with sums in 32 bits (fp32 numbers as sums of three bf16 ones, so that nothing of them
    is lost; an infinity among them gives NaN).  In bf16 and fp16 the hidden vectors and the gradients of the two projections are rounded to
    that type, as the tensor cores read them: one rounding beside that of the results, and in fp16 an infinity where one of them passes 65504.  For the
    backward a call keeps the hidden vectors and, in 32 bits, their derivatives by the two projections: 10 bytes a hidden value, in fp32 14.  ``x``
    and weights whose rows are not runs of consecutive elements (a weight that is another's transpose) or do not begin on 16-byte boundaries, and those in
    fp32, are copied in each call."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"flex_rnn_b200: gated_mlp: activation has to be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    _operators()
    return _ops.gated_mlp.default(x, gate, up, down, ACTIVATIONS.index(activation), False)[0]


def rotary(x: th.Tensor, positions: Union[int, th.Tensor], frequencies: th.Tensor, interleaved: bool = False, scale: float = 1.0) -> th.Tensor:
    """Rotary positions on ``x`` [batch, length, ..., width], for instance the queries and keys [B,T,H,1,N] of a scan: of the
    first ``2 * len(frequencies)`` values of each head, pairs (u, w) become ``scale * (u cos - w sin, u sin + w cos)``
    with the angle ``position * frequency``; the other values are copied.

    ``positions`` is [length] or [batch, length] in int64 or int32, or a number: the first place's position, the others follow.
    ``frequencies`` (fp32 or fp64, see ``rotary_frequencies``) are radians a position.  Pair i is (i, i + pairs), or
    (2 i, 2 i + 1) with ``interleaved``.  Angles are computed in 64 bits: far positions lose nothing.  The result is contiguous.
    Differentiable in ``x``, also more than once."""
    _operators()
    start, where = (0, positions) if isinstance(positions, th.Tensor) else (positions, None)
    return _ops.rotary.default(x, where, start, frequencies, interleaved, scale, False)


def rotary_frequencies(width: int, base: float = 10000.0, factor: float = 1.0, method: str = "linear", length: Optional[int] = None, turns=(1.0, 32.0), device=None) -> th.Tensor:
    """Frequencies of ``width / 2`` pairs, ``base ** (-2 i / width)``, in fp64, for ``rotary``; ``width`` is the number of values
    that are turned, at most a head's.

    For contexts ``factor`` times as long as those of training: ``method="linear"`` divides all of them by ``factor``;
    ``"base"`` multiplies the base by ``factor ** (width / (width - 2))``, so that the first stays and the last is divided by
    ``factor``; ``"parts"`` divides those that make fewer than ``turns[0]`` turns within the ``length`` of training, keeps those
    that make more than ``turns[1]``, and goes linearly from the one to the other between them (``scale`` of ``rotary`` is then
    usually ``0.1 * log(factor) + 1``)."""
    if width < 0 or width % 2:
        raise ValueError(f"flex_rnn_b200: rotary_frequencies: width has to be even, got {width}")
    if not (base > 0 and factor > 0):
        raise ValueError(f"flex_rnn_b200: rotary_frequencies: base and factor have to be positive, got {base} and {factor}")
    if method == "base" and width > 2:
        base = base * factor ** (width / (width - 2))
    f = base ** (-th.arange(0, width, 2, dtype=th.float64, device=device) / max(width, 1))
    if method == "linear":
        return f / factor
    if method == "base":
        return f
    if method != "parts":
        raise ValueError(f"flex_rnn_b200: rotary_frequencies: method has to be linear, base or parts, got {method!r}")
    if length is None or not turns[0] < turns[1]:
        raise ValueError("flex_rnn_b200: rotary_frequencies: parts needs the length of training, and turns in rising order")
    keep = ((length * f / (2 * math.pi) - turns[0]) / (turns[1] - turns[0])).clamp(0, 1)
    return f * keep + f / factor * (1 - keep)


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


def naive_linear_logprobs(x, weight, tokens, temperature=1.0, ignore_index=-100):
    """Definition of ``linear_logprobs`` in the arithmetic of ``x``."""
    return LinearLogprobs(*naive_token_logprobs(x @ weight.t(), tokens, 0, temperature, ignore_index)[:2])


def naive_gated_mlp(x, gate, up, down, activation="silu"):
    """Definition of ``gated_mlp`` in the arithmetic of ``x``."""
    act = {"silu": th.nn.functional.silu, "gelu": th.nn.functional.gelu, "relu": th.relu, "sigmoid": th.sigmoid}[activation]
    return (act(x @ gate.t()) * (x @ up.t())) @ down.t()


def naive_rotary(x, positions, frequencies, interleaved=False, scale=1.0):
    """Definition of ``rotary`` in the arithmetic of ``x``, with angles in 64 bits."""
    if not isinstance(positions, th.Tensor):
        positions = positions + th.arange(x.shape[1], device=x.device)
    angle = positions.double()[..., None] * frequencies
    angle = angle.view(*(1,) * (3 - angle.dim()), *angle.shape[:-1], *(1,) * (x.dim() - 3), -1)
    cos, sin = (scale * angle.cos()).to(x.dtype), (scale * angle.sin()).to(x.dtype)
    pairs = frequencies.shape[0]
    u, w = (x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]) if interleaved else (x[..., :pairs], x[..., pairs:2 * pairs])
    turned = (u * cos - w * sin, u * sin + w * cos)
    turned = th.stack(turned, -1).flatten(-2) if interleaved else th.cat(turned, -1)
    return th.cat([turned, x[..., 2 * pairs:]], -1)


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

    @fake("flex_rnn_b200::linear_logprobs")
    def _(x, weight, tokens, temperature, ignore_index, save):
        new = lambda *shape: x.new_empty(shape, dtype=th.float32)
        return new(*tokens.shape), new(*tokens.shape), new(tokens.numel() if save else 0, 2)

    @fake("flex_rnn_b200::linear_logprobs_backward")
    def _(dlogprob, dentropy, x, weight, tokens, stats, temperature, ignore_index, want_x, want_weight):
        return x.new_empty(x.shape if want_x else (0,)), x.new_empty(weight.shape if want_weight else (0,))

    @fake("flex_rnn_b200::gated_mlp")
    def _(x, gate, up, down, activation, save):
        kept = (x.numel() // x.shape[-1] if save else 0, (gate.shape[0] + 63) // 64 * 64)
        hidden = x.new_empty((3, *kept), dtype=th.bfloat16) if x.dtype == th.float32 else x.new_empty((1, *kept))
        by = x.new_empty((2, *kept), dtype=th.float32)
        return x.new_empty((*x.shape[:-1], down.shape[0])), by[0].clone(), by[1].clone(), hidden

    @fake("flex_rnn_b200::gated_mlp_backward")
    def _(grad, x, gate, up, down, by_gate, by_up, hidden, activation, want_x, want_gate, want_up, want_down):
        return tuple(x.new_empty(t.shape if want else (0,)) for t, want in ((x, want_x), (gate, want_gate), (up, want_up), (down, want_down)))

    @fake("flex_rnn_b200::rotary")
    def _(x, positions, start, frequencies, interleaved, scale, inverse):
        return x.new_empty(x.shape)
