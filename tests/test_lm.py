"""The operators around the scans (flex_rnn_b200.lm) against their definitions in 64 bits.

Tolerances: a result of type t is the exact one rounded once (relative 2^-24 for fp32, 2^-11 for fp16, 2^-8 for bf16: half
a unit of the last place of the smallest mantissa), plus the error of arithmetic in 32 bits.  n additions of rounding
2^-24 go astray by about sqrt(n) 2^-24 of the sum of the terms' absolute values; 64 covers 4096 additions in a row, which
no thread makes.  ``near`` takes that sum of absolute values (of a formula: of all its terms, with what their own inputs
lost) as ``size``."""
import contextlib
import ctypes
import math

import pytest
import torch

import flex_rnn_b200 as fr
from flex_rnn_b200 import lm, runtime

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def near(got, want, size):
    """Everywhere within one rounding and the error of 32-bit sums whose terms' absolute values add up to ``size``."""
    assert got.shape == want.shape
    g, w = got.detach().double().cpu(), want.detach().double().cpu()
    size = torch.as_tensor(size, dtype=torch.float64).detach().cpu().expand(w.shape)
    assert torch.equal(g.isnan(), w.isnan())
    far = torch.isinf(w)
    assert torch.equal(g[far], w[far])
    fine = torch.isfinite(w)
    tol = UNIT[got.dtype] * w.abs() + 64 * 2.0 ** -24 * size + TINY[got.dtype]
    off = ((g - w).abs() - tol)[fine]
    assert not off.numel() or off.max() <= 0, f"{int((off > 0).sum())} of {off.numel()} values off, worst by {float(off.max())} over the tolerance"


def rand(*shape, seed=0, device="cuda"):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape)), dtype=torch.float32).to(device)


def off_boundary(t):
    """The values of ``t``, contiguous, one element off a 16-byte boundary."""
    return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)


# ---- embedding -------------------------------------------------------------------------------------------------------------

def embedding_case(n, V, D, dtype, seed=0, pad=False, same=False, token_dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(0, V, (n,), generator=g)
    if same:
        t[:] = V - 1
        t[: n // 7] = torch.randint(0, V, (n // 7,), generator=g)
    if pad:
        t[torch.rand(n, generator=g) < 0.3] = -100
    return t.to(token_dtype).cuda(), rand(V, D, seed=seed).to(dtype), rand(n, D, seed=seed + 1).to(dtype)


def embedding_check(t, w, dy, scale=1.0, ignore=-100):
    leaf = w.detach().requires_grad_()
    y = fr.embedding(t, leaf, scale=scale, ignore_index=ignore)
    (dw,) = torch.autograd.grad(y, leaf, dy)
    assert y.dtype == dw.dtype == w.dtype and y.is_contiguous()
    exact = w.detach().double().requires_grad_()
    want = lm.naive_embedding(t.long(), exact, scale, ignore)
    near(y, want, want.abs())
    there = (t != ignore).reshape(-1)
    at, d = t.reshape(-1).long()[there], dy.double().reshape(-1, w.shape[1])[there] * scale
    zero = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
    near(dw, zero.index_add(0, at, d), zero.index_add(0, at, d.abs()))
    return y, dw


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (1, 65536, 512), (3, 2, 7), (37, 100, 64), (257, 1000, 96), (700, 313, 515), (2048, 256, 256), (1500, 70001, 33),
                                   (5000, 9, 130), (64, 300000, 24), (4097, 5003, 1028)])
def test_embedding(n, V, D, dtype):
    embedding_check(*embedding_case(n, V, D, dtype), scale=D ** 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,D,same,pad", [(5000, 700, 72, True, False), (5000, 700, 72, False, True), (3001, 50, 17, True, True), (20000, 3, 8, True, False),
                                            (40000, 70000, 40, True, True), (70, 1, 2056, False, True)])
def test_embedding_of_one_token_and_padding(n, V, D, same, pad, dtype):
    """One token in most places (its row's sum is long), padded places, both."""
    embedding_check(*embedding_case(n, V, D, dtype, same=same, pad=pad), scale=0.5)


@pytest.mark.gpu
def test_embedding_layouts():
    t, w, dy = embedding_case(96, 211, 48, torch.bfloat16, token_dtype=torch.int32)
    for weight in (w, w.t().contiguous().t(), off_boundary(w), rand(211, 80, seed=5).bfloat16()[:, 8:56], rand(211, 80, seed=5).bfloat16()[:, 3:51],
                   rand(422, 48, seed=6).bfloat16()[::2], rand(1, 48).bfloat16().expand(211, 48)):
        for tokens, up in ((t.view(2, 48), dy.view(2, 48, 48)), (t.view(48, 2).t(), dy.view(2, 48, 48)), (t.view(4, 2, 12), off_boundary(dy).view(4, 2, 12, 48)),
                           (t.view(2, 48), dy[:1].expand(96, 48).view(2, 48, 48)), (t.view(2, 48), dy.view(2, 48, 48).transpose(0, 1).contiguous().transpose(0, 1))):
            embedding_check(tokens, weight, up, scale=-3.0)
    embedding_check(t[5], w, dy[5])                                              # one token without a dimension
    t[::3] = -1
    embedding_check(t, w, dy, ignore=-1)
    embedding_check(torch.full_like(t, -100), w, dy)                             # nothing but padding


@pytest.mark.gpu
def test_embedding_empty():
    w = rand(11, 5).requires_grad_()
    y = fr.embedding(torch.empty(0, 3, dtype=torch.int64, device="cuda"), w)
    assert y.shape == (0, 3, 5) and torch.equal(torch.autograd.grad(y.sum(), w)[0], torch.zeros_like(w))
    w0 = torch.empty(4, 0, device="cuda", requires_grad=True)
    y = fr.embedding(torch.tensor([1, 3], device="cuda"), w0)
    assert y.shape == (2, 0) and torch.autograd.grad(y.sum(), w0)[0].shape == (4, 0)


@pytest.mark.gpu
def test_embedding_token_outside_the_vocabulary():
    """Zeros and no gradient at that place; the next call raises, the one after it runs."""
    w = rand(11, 16).requires_grad_()
    for bad in (11, -1, 2 ** 31 + 1, -2 ** 40):
        t = torch.tensor([3, bad, 3], device="cuda")
        y = fr.embedding(t, w)
        torch.cuda.synchronize()
        assert not y[1].any() and torch.equal(y[0], w[3])
        with pytest.raises(runtime.FrnnError, match="outside the vocabulary"):
            fr.embedding(t[:1], w)
        g = torch.autograd.grad(y, w, torch.ones_like(y))[0]
        assert float(g.sum()) == 32.0 and float(g[3, 0]) == 2.0
        assert torch.equal(fr.embedding(t[:1], w)[0], w[3])


@pytest.mark.gpu
def test_embedding_offsets_past_31_bits():
    V, D = 70001, 32768                             # 2.29e9 elements
    w = torch.zeros(V, D, dtype=torch.bfloat16, device="cuda")
    w[V - 1] = rand(D).bfloat16()
    w[40000] = 2.0
    w.requires_grad_()
    t = torch.tensor([V - 1, 40000, V - 1, 0], device="cuda")
    y = fr.embedding(t, w)
    assert torch.equal(y[0], w[V - 1]) and torch.equal(y[2], y[0]) and bool((y[1] == 2).all()) and not y[3].any()
    (g,) = torch.autograd.grad(y, w, torch.ones_like(y))
    sums = g.sum(1, dtype=torch.float32)
    assert float(sums[V - 1]) == 2 * D and float(sums[40000]) == D and float(sums[0]) == D and float(sums.sum()) == 4 * D


# ---- layer norm ------------------------------------------------------------------------------------------------------------

def layer_norm_check(x, w, b, dy, eps=1e-5):
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = fr.layer_norm(*leaves, eps=eps)
    assert y.dtype == x.dtype and y.is_contiguous() and y.shape == x.shape
    got = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    assert got[0].stride() == torch.empty_like(x).stride()
    exact = [None if t is None else t.detach().double().requires_grad_() for t in (x, w, b)]
    want_y = lm.naive_layer_norm(*exact, eps=eps)
    want = torch.autograd.grad(want_y, [t for t in exact if t is not None], dy.double())
    xd, g = exact[0].detach(), dy.double()
    one = torch.ones((), dtype=torch.float64, device=x.device)
    wd, bd = (one if t is None else t.detach().abs() for t in exact[1:])
    mean = xd.mean(-1, True)
    rstd = ((xd - mean).square().mean(-1, True) + eps).rsqrt()
    xh = ((xd - mean) * rstd).abs() + (xd.abs() + mean.abs()) * rstd          # with what the subtraction of the mean loses
    near(y, want_y, xh * wd + (bd if b is not None else 0.0))
    gw = g.abs() * wd
    near(got[0], want[0], rstd * (gw + gw.mean(-1, True) + xh * (gw * xh).mean(-1, True)))
    over = tuple(range(x.dim() - w.dim())) if w is not None else None
    if w is not None:
        near(got[1], want[1], (g.abs() * xh).sum(over))
    if b is not None:
        near(got[-1], want[-1], g.abs().sum(over if over is not None else tuple(range(x.dim() - b.dim()))))
    return (y, *got)


def params(kind, H, D, dtype):
    shape = {"vector": (D,), "heads": (H, D), "none": None}[kind]
    return (None, None) if shape is None else ((1 + 0.2 * rand(*shape, seed=3)).to(dtype), (0.3 * rand(*shape, seed=4)).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("io,par", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
@pytest.mark.parametrize("rows,D", [(1, 1), (1, 2), (5, 8), (1, 4096), (33, 31), (300, 64), (7, 100), (130, 257), (64, 1000), (61, 1001), (40, 1024), (17, 2500),
                                    (9, 4095), (12, 8192), (3, 8200), (2, 16384), (2, 40001), (2000, 16)])
def test_layer_norm(rows, D, io, par):
    x, dy = (0.4 + rand(rows, D)).to(io), rand(rows, D, seed=2).to(io)
    layer_norm_check(x, *params("vector", 1, D, par), dy)


@pytest.mark.gpu
@pytest.mark.parametrize("io,par", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("kind", ["heads", "vector", "none"])
@pytest.mark.parametrize("B,T,H,D", [(2, 5, 3, 64), (1, 1, 32, 128), (3, 7, 1, 64), (2, 33, 5, 96), (1, 50, 4, 77), (2, 3, 24, 16), (1, 4, 2, 1500), (1, 300, 7, 130)])
def test_layer_norm_of_heads(B, T, H, D, kind, io, par):
    x, dy = (rand(B, T, H, D) - 0.2).to(io), rand(B, T, H, D, seed=2).to(io)
    layer_norm_check(x, *params(kind, H, D, par), dy)


@pytest.mark.gpu
@pytest.mark.parametrize("io,par", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("rows,H,D", [(700, 1, 601), (90, 3, 1016), (350, 1, 1801), (30, 2, 2040), (310, 1, 3601), (20, 2, 4088), (9, 3, 1100), (300, 1, 2561), (5, 2, 6001)])
def test_layer_norm_of_several_warps(rows, H, D, io, par):
    """Rows of more than one warp: whole blocks and groups of 64, 128 and 256 lanes, even, odd and sliced, more rows than groups."""
    w, b = params("heads" if H > 1 else "vector", H, D, par)
    x, dy = (0.5 + rand(rows, H, D)).to(io), rand(rows, H, D, seed=2).to(io)
    layer_norm_check(x, w, b, dy)
    layer_norm_check((rand(rows, H, D + 5, seed=6) - 0.5).to(io)[..., 5:], w, b, dy)
    layer_norm_check(x.view(rows * H, D), *params("vector", 1, D, par), dy.view(rows * H, D))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["heads", "vector"])
def test_layer_norm_layouts(kind):
    B, T, H, D = 2, 6, 3, 64
    dy0 = rand(B, T, H, D, seed=2).bfloat16()
    w, b = params(kind, H, D, torch.bfloat16)
    flat = lambda *s: rand(*s, seed=7).bfloat16()
    xs = [flat(B, T, 3, H, D)[:, :, 1], flat(B, H, T, D).transpose(1, 2), flat(B, T, H, D + 8)[..., 8:], flat(B, T, H, D + 3)[..., 3:], flat(B, T, D, H).transpose(2, 3),
          off_boundary(flat(B, T, H, D)), flat(B, T, 1, D).expand(B, T, H, D), flat(1, 1, H, D).expand(B, T, H, D), flat(B, T, H, 1).expand(B, T, H, D),
          flat(H, T, B, D).permute(2, 1, 0, 3), flat(2 * B, T, H, D)[::2], flat(B, 2 * T, 2 * H, D)[:, ::2, ::2]]
    dys = [dy0, off_boundary(dy0), dy0[..., :1].expand(B, T, H, D), dy0.transpose(1, 2).contiguous().transpose(1, 2), dy0[:1, :1].expand(B, T, H, D)]
    for x in xs:
        layer_norm_check(x, w, b, dy0)
    for dy in dys:
        layer_norm_check(xs[0], w, b, dy)
    layer_norm_check(xs[0], w, None, dy0)
    layer_norm_check(xs[0], None, b, dy0)
    layer_norm_check(xs[0], rand(2 * D, seed=3).bfloat16()[::2] if kind == "vector" else rand(D, H, seed=3).bfloat16().t(), None, dy0)
    layer_norm_check(xs[0], off_boundary(w), off_boundary(b), dy0)
    six = flat(2, 3, 2, 2, H, D).permute(3, 1, 0, 2, 4, 5)                    # five strides between rows: copied
    layer_norm_check(six, w, b, flat(2, 3, 2, 2, H, D))
    if kind == "vector":
        layer_norm_check(flat(D), w, b, rand(D, seed=9).bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("D", [40, 4096])
def test_layer_norm_of_difficult_rows(D):
    """Constant rows, a mean far from zero, very small and very large values; NaN and infinity stay in their row."""
    w, b = params("vector", 1, D, torch.float32)
    x = rand(6, D)
    x[0], x[1], x[2], x[3], x[4] = 3.0, 1000 + x[1], 1e-6 * x[2], 1e6 * x[3], 0.0
    layer_norm_check(x, w, b, rand(6, D, seed=2))
    assert torch.equal(fr.layer_norm(x, w, b)[4], b)
    x[1, 3], x[5, 7] = math.nan, math.inf
    leaf = x.clone().requires_grad_()
    y = fr.layer_norm(leaf, w, b)
    g = torch.autograd.grad(y, leaf, torch.ones_like(y))[0]
    for t in (y, g):
        assert t[[1, 5]].isnan().all() and t[[0, 2, 3, 4]].isfinite().all()


@pytest.mark.gpu
def test_layer_norm_empty():
    w = rand(8).requires_grad_()
    b = rand(8, seed=1).requires_grad_()
    x = torch.empty(0, 8, device="cuda", requires_grad=True)
    y = fr.layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == gx.shape == (0, 8) and not gw.any() and not gb.any()
    x = torch.empty(3, 0, device="cuda", requires_grad=True)
    assert torch.autograd.grad(fr.layer_norm(x).sum(), x)[0].shape == (3, 0)


@pytest.mark.gpu
def test_layer_norm_offsets_past_31_bits():
    R, D = 131100, 16384                            # 2.15e9 elements
    x = torch.zeros(R, D, dtype=torch.bfloat16, device="cuda")
    x[-1], x[R // 2] = rand(D).bfloat16(), rand(D, seed=1).bfloat16()
    w = (1 + 0.2 * rand(D, seed=3)).requires_grad_()
    leaf = x.requires_grad_()
    y = fr.layer_norm(leaf, w)
    rows = [R - 1, R // 2, 5]
    want = lm.naive_layer_norm(x.detach()[rows].double(), w.detach().double())
    near(y[rows], want, want.abs() + 1)
    dy = torch.zeros_like(x)
    dy[-1] = rand(D, seed=2).bfloat16()
    gx, gw = torch.autograd.grad(y, (leaf, w), dy)
    last, wd = x.detach()[-1:].double().requires_grad_(), w.detach().double().requires_grad_()
    ex, ew = torch.autograd.grad(lm.naive_layer_norm(last, wd), (last, wd), dy[-1:].double())
    near(gx[-1:], ex, 4.0 * (1 + dy[-1:].double().abs()))
    near(gw, ew, 4.0 * dy[-1].double().abs())
    assert not gx[:-1].any()


# ---- log probabilities ---------------------------------------------------------------------------------------------------------

def logprobs_check(logits, tokens, top=0, temperature=1.0, ignore=-100, up=None):
    leaf = logits.detach().requires_grad_()
    r = fr.token_logprobs(leaf, tokens, top=top, temperature=temperature, ignore_index=ignore)
    assert r.logprob.dtype == r.entropy.dtype == r.top_logprob.dtype == torch.float32 and r.top_token.dtype == torch.int64
    assert not r.top_logprob.requires_grad
    exact = logits.detach().double().requires_grad_()
    want = lm.naive_token_logprobs(exact, tokens.long(), top, temperature, ignore)
    z = logits.double() / temperature
    none = (logits == -math.inf).all(-1)
    logp = torch.log_softmax(torch.where(none[..., None], 0.0, z), -1)
    p = torch.where(none[..., None], 0.0, logp.exp())
    lost = 1 + torch.where(p > 0, -logp, 0.0)                                   # an exponent's rounding, relative to its result
    rounded = lambda t: torch.where(t.isfinite(), t.abs(), 0.0) / 8              # eight roundings relative to the result
    near(r.logprob, want.logprob, 1 + rounded(want.logprob))
    near(r.entropy, want.entropy, (p * lost * lost).sum(-1) + 1)
    assert torch.equal(r.top_token, want.top_token)
    near(r.top_logprob, want.top_logprob, 1 + rounded(want.top_logprob))
    up = up or (rand(*tokens.shape, 1, seed=11)[..., 0], rand(*tokens.shape, 1, seed=12)[..., 0])
    g = torch.autograd.grad((r.logprob, r.entropy), leaf, up)[0]
    assert g.dtype == logits.dtype and g.shape == logits.shape
    # by the formula: rows without any token, whose log probabilities autograd cannot pass, have gradient 0
    there = (tokens != ignore)
    glp, gh = torch.where(there, up[0].double(), 0.0)[..., None], up[1].double()[..., None]
    H = want.entropy.detach()[..., None]
    lp = torch.where(p > 0, logp, 0.0)
    hit = torch.zeros_like(p).scatter_(-1, torch.where(there, tokens, 0).long()[..., None], 1.0)
    d = torch.where(none[..., None], 0.0, (glp * (hit - p) - gh * p * (lp + H)) / temperature)
    size = (glp.abs() * (hit + p * lost) + gh.abs() * p * lost * (lp.abs() + H + 1)) / temperature
    near(g, d, torch.where(none[..., None], 0.0, size))
    return r, g


def logits_of(n, V, dtype, seed=0, spread=2.0):
    return (spread * rand(n, V, seed=seed)).to(dtype), torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,top", [(1, 1, 1), (1, 2, 2), (3, 5, 5), (1, 65536, 20), (16, 65536, 32), (7, 1000, 3), (200, 313, 8), (33, 32003, 5), (2, 200001, 32), (5, 33, 32),
                                     (300, 4096, 0), (1000, 520, 1), (2, 40, 31)])
def test_token_logprobs(n, V, top, dtype):
    logprobs_check(*logits_of(n, V, dtype), top=top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature", [0.3, 1.7, 25.0])
def test_token_logprobs_temperature(temperature, dtype):
    logprobs_check(*logits_of(9, 777, dtype), top=4, temperature=temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [40, 3001, 70000])
def test_token_logprobs_masks(V, dtype):
    """Masked by -inf and by the type's lowest value: most of a row, all of it, all but one, the token itself; padding."""
    x, t = logits_of(12, V, dtype)
    lowest = torch.finfo(dtype).min
    keep = torch.rand(12, V, generator=torch.Generator().manual_seed(3)).cuda() < 0.1
    keep.scatter_(1, t[:, None], True)
    x = torch.where(keep, x, -math.inf)
    x[0] = -math.inf
    x[1] = lowest
    x[2] = -math.inf
    x[2, V - 1] = 0.7
    x[3, t[3]] = -math.inf                    # a token that may not follow
    x[4] = torch.where(keep[4], x[4], lowest)
    x[5] = torch.where(keep[5], x[5], lowest)
    x[5, t[5]] = lowest
    x[6] = lowest
    x[6, V // 2] = -math.inf
    t[7] = -100
    t[0 if V == 40 else 8] = -100
    x[9] = 0.0
    x[10, t[10]] = torch.finfo(dtype).max / 4
    logprobs_check(x, t, top=min(V, 32))


@pytest.mark.gpu
def test_token_logprobs_ties():
    """Equal logits come by the lowest token, wherever they lie in the row; -0 equals 0."""
    for V in (32, 1000, 9001, 66000):
        x = torch.zeros(5, V, device="cuda", dtype=torch.bfloat16)
        x[1, ::2] = -0.0
        x[2] = (torch.arange(V, device="cuda") % 7).bfloat16()
        x[3, V // 2:] = 1.0
        x[4] = -torch.arange(V, device="cuda").float().div(300).floor().bfloat16()
        logprobs_check(x, torch.arange(5, device="cuda"), top=32)
        x = torch.arange(V, device="cuda").float().expand(2, V) * 1e-3           # ever larger: each is the best so far
        logprobs_check(x, torch.tensor([0, V - 1], device="cuda"), top=32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_token_logprobs_nan_and_infinity(dtype):
    """NaN or +inf make their row NaN and leave the others alone."""
    x, t = logits_of(6, 1001, dtype)
    clean, gc = logprobs_check(x, t)
    x[1, 500], x[2, 3], x[4, t[4]] = math.nan, math.inf, math.inf
    leaf = x.requires_grad_()
    r = fr.token_logprobs(leaf, t, top=3)
    g = torch.autograd.grad((r.logprob, r.entropy), leaf, (torch.ones(6, device="cuda"), torch.ones(6, device="cuda")))[0]
    for i in range(6):
        bad = i in (1, 2, 4)
        assert bool(r.logprob[i].isnan()) == bad and bool(r.entropy[i].isnan()) == bad and bool(r.top_logprob[i].isnan().all()) == bad and bool(g[i].isnan().all()) == bad
        assert bad or (r.logprob[i] == clean.logprob[i] and g[i].isfinite().all())
    assert r.top_token[1, 0] == 500 and r.top_token[2, 0] == 3 and r.top_token[4, 0] == t[4]


@pytest.mark.gpu
def test_token_logprobs_layouts():
    x, t = logits_of(24, 350, torch.bfloat16)
    logprobs_check(x.view(2, 3, 4, 350), t.view(2, 3, 4), top=5)
    logprobs_check(x.view(2, 12, 350).transpose(0, 1), t.view(2, 12).t(), top=5)
    logprobs_check(rand(24, 400).bfloat16()[:, 8:358], t.int(), top=5)
    logprobs_check(rand(24, 401).bfloat16()[:, 3:353], t, top=5)
    logprobs_check(rand(350, 24).bfloat16().t(), t, top=5)
    logprobs_check(off_boundary(x), t, top=5)
    logprobs_check(x[:1].expand(24, 350), t, top=5)
    logprobs_check(x[::2], t[::2], top=5, ignore=int(t[4]))
    logprobs_check(x[3], t[3], top=5)
    logprobs_check(x, t, up=(torch.ones((), device="cuda").expand(24), rand(24, 2)[:, 1]))
    empty = torch.empty(0, 350, device="cuda", requires_grad=True)
    r = fr.token_logprobs(empty, t[:0], top=2)
    assert r.logprob.shape == (0,) and r.top_token.shape == (0, 2) and torch.autograd.grad(r.entropy.sum(), empty)[0].shape == (0, 350)


@pytest.mark.gpu
def test_token_logprobs_single_outputs():
    """The gradient of one output alone."""
    x, t = logits_of(6, 500, torch.float32)
    zero, up = torch.zeros(6, device="cuda"), rand(6)
    _, a = logprobs_check(x, t, up=(up, zero))
    _, b = logprobs_check(x, t, up=(zero, up))
    leaf = x.requires_grad_()
    r = fr.token_logprobs(leaf, t, top=1)
    assert torch.equal(torch.autograd.grad(r.logprob, leaf, up, retain_graph=True)[0], a)
    assert torch.equal(torch.autograd.grad(r.entropy, leaf, up)[0], b)


@pytest.mark.gpu
def test_token_logprobs_token_outside_the_vocabulary():
    x, t = logits_of(4, 60, torch.float32)
    for bad in (60, -7, 2 ** 33):
        u = t.clone()
        u[2] = bad
        leaf = x.clone().requires_grad_()
        r = fr.token_logprobs(leaf, u)
        torch.cuda.synchronize()
        assert r.logprob.isnan().tolist() == [False, False, True, False]
        with pytest.raises(runtime.FrnnError, match="outside the vocabulary"):
            fr.token_logprobs(leaf, t)
        assert torch.autograd.grad(r.logprob, leaf, torch.ones(4, device="cuda"))[0].isfinite().all()


@pytest.mark.gpu
def test_token_logprobs_offsets_past_31_bits():
    n, V = 16500, 131072                            # 2.16e9 elements
    x = torch.zeros(n, V, dtype=torch.bfloat16, device="cuda")
    x[-1] = rand(V).bfloat16()
    t = torch.full((n,), 17, device="cuda")
    leaf = x.requires_grad_()
    r = fr.token_logprobs(leaf, t, top=3)
    want = lm.naive_token_logprobs(x.detach()[-1:].double(), t[-1:], top=3)
    near(r.logprob[-1:], want.logprob, 16.0)
    assert torch.equal(r.top_token[-1:], want.top_token) and r.top_token[-2].tolist() == [0, 1, 2]
    near(r.logprob[:-1], torch.full((n - 1,), -math.log(V), dtype=torch.float64), 16.0)
    g = torch.autograd.grad(r.logprob.sum(), leaf)[0]
    near(g[-1], torch.nn.functional.one_hot(t[-1], V).double().cpu() - torch.softmax(x.detach()[-1].double(), -1).cpu(), 1.0 / V)
    assert bool((g[:-1, 18:] == g[0, 18]).all())


# ---- all of them ----------------------------------------------------------------------------------------------------------------

def calls(dtype=torch.float32):
    """name -> (function of its leaves, the leaves, upstream gradients)"""
    t = torch.randint(0, 50, (3, 20), generator=torch.Generator().manual_seed(1)).cuda()
    w, x, z = rand(50, 48), rand(3, 20, 4, 16), rand(3, 20, 50)
    g, b = 1 + 0.1 * rand(4, 16, seed=1), rand(4, 16, seed=2)
    one = lambda f: lambda *a: (f(*a),)
    out = {"embedding": (one(lambda w: fr.embedding(t, w, scale=1.5)), [w], [rand(3, 20, 48, seed=5)]),
           "layer_norm": (one(fr.layer_norm), [x, g, b], [rand(3, 20, 4, 16, seed=6)]),
           "token_logprobs": (lambda z: fr.token_logprobs(z, t, temperature=0.9)[:2], [z], [rand(3, 20, seed=7), rand(3, 20, seed=8)])}
    return {k: (f, [v.to(dtype).requires_grad_() for v in a], [u if k == "token_logprobs" else u.to(dtype) for u in up]) for k, (f, a, up) in out.items()}


def both(f, leaves, up, ctx=contextlib.nullcontext()):
    with ctx:
        y = f(*leaves)
    return [*(v.detach() for v in y), *torch.autograd.grad(y, leaves, up)]


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["embedding", "layer_norm", "token_logprobs"])
def test_gradients_against_differences(name):
    """Central differences of the operator's own forward along random directions, in fp32.  Truncation: the third
    derivative along d is at most about 10 (values of order 1), times h^2 / 6; rounding: 2^-24 of each output, in random
    directions, over 2 h."""
    f, leaves, up = calls()[name]
    grads = torch.autograd.grad(f(*leaves), leaves, up)
    h = 2.0 ** -6
    value = lambda a: [y.double() for y in f(*a)]
    for i, (leaf, g) in enumerate(zip(leaves, grads)):
        for seed in range(3):
            d = rand(*leaf.shape, seed=40 + seed)
            d = d / d.norm() * 8
            step = lambda s: [v.detach() + (s * d if j == i else 0) for j, v in enumerate(leaves)]
            hi, lo = value(step(h)), value(step(-h))
            diff = sum(float(((a - b) * u.double()).sum()) for a, b, u in zip(hi, lo, up)) / (2 * h)
            size = sum(float(u.double().norm() * a.norm()) for a, u in zip(hi, up))
            bend = 10 * float(d.abs().max()) ** 2 * sum(float(u.double().norm()) for u in up) * 8
            assert abs(diff - float((g.double() * d.double()).sum())) <= 4 * 2.0 ** -24 * size / (2 * h) + bend * h * h / 6


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["embedding", "layer_norm", "token_logprobs"])
def test_repeated_calls_give_the_same_bits(name):
    f, leaves, up = calls(torch.bfloat16)[name]
    want = both(f, leaves, up)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(both(f, leaves, up), want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["embedding", "layer_norm", "token_logprobs"])
def test_streams_graphs_and_threads(name):
    f, leaves, up = calls()[name]
    want = both(f, leaves, up)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        got = both(f, leaves, up)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    still = [v.detach().clone().zero_().requires_grad_() for v in leaves]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both(f, still, up)
    with torch.no_grad():
        for a, b in zip(still, leaves):
            a.copy_(b)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["embedding", "layer_norm", "token_logprobs"])
def test_compiled(name):
    f, leaves, up = calls()[name]
    compiled = torch.compile(lambda *a: tuple(2 * v for v in f(*a)), fullgraph=True, dynamic=False)
    plain = lambda *a: tuple(2 * v for v in f(*a))
    for a, b in zip(both(compiled, leaves, up), both(plain, leaves, up)):
        assert a.dtype == b.dtype and torch.equal(a, b)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(compiled(*leaves), plain(*leaves)))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["embedding", "layer_norm", "token_logprobs"])
def test_graph_semantics(name):
    """Second use, changed inputs, saved-tensor hooks, batched upstream gradients, gradients of gradients."""
    f, leaves, up = calls()[name]
    want = both(f, leaves, up)[-len(leaves):]
    y = f(*leaves)
    first = torch.autograd.grad(y, leaves, up, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, want))
    up = [u.requires_grad_() for u in up]         # (the gradient of an embedding depends on nothing else)
    first = torch.autograd.grad(f(*leaves), leaves, up, create_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(first[0].sum(), up[0])
    if name != "embedding":
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(torch.autograd.grad(f(*leaves), leaves, [u.detach() for u in up], create_graph=True)[0].sum(), leaves[0])
    up = [u.detach() for u in up]
    y = f(*leaves)
    torch.autograd.grad(y, leaves, up)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, leaves, up)
    hooks = torch.autograd.graph.saved_tensors_hooks
    for ctx in (torch.autograd.graph.save_on_cpu(pin_memory=True), hooks(off_boundary, lambda t: t), hooks(lambda t: t.t().contiguous() if t.dim() == 2 else t, lambda t: t.t() if t.dim() == 2 else t)):
        assert all(torch.equal(a, b) for a, b in zip(both(f, leaves, up, ctx)[-len(leaves):], want))
    y = f(*leaves)
    many = torch.autograd.grad(y, leaves, [torch.stack([u, -2 * u]) for u in up], is_grads_batched=True)
    for a, b in zip(many, want):
        assert torch.equal(a[0], b) and torch.equal(a[1], -2 * b)
    if name != "embedding":
        y = f(*leaves)
        with torch.no_grad():
            leaves[0].add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, leaves, up)


@pytest.mark.gpu
def test_guard_bands_and_checked_calls(monkeypatch):
    """With FRNN_GUARD=1 no kernel writes outside of its buffers, at sizes that end inside of accesses, tiles and chunks;
    with FRNN_CHECK=1 a call raises what its own kernels reported."""
    monkeypatch.setenv("FRNN_GUARD", "1")
    for dtype in DTYPES:
        for n, V, D in [(1, 3, 1), (37, 100, 64), (301, 50, 77), (700, 2003, 515), (3000, 70, 1030), (5000, 300, 33)]:
            embedding_check(*embedding_case(n, V, D, dtype, pad=n % 2 == 1, same=n == 5000))
        for rows, H, D in [(1, 1, 1), (5, 1, 31), (40, 3, 77), (33, 5, 128), (130, 1, 1001), (61, 1, 2047), (9, 1, 4096), (5, 1, 8200)]:
            x, dy = rand(rows, H, D).to(dtype), rand(rows, H, D, seed=2).to(dtype)
            layer_norm_check(x, *params("heads" if H > 1 else "vector", H, D, dtype), dy)
            layer_norm_check(rand(rows, H, D + 3, seed=4).to(dtype)[..., 3:], *params("vector", H, D, torch.float32), dy)
        for n, V, top in [(1, 1, 1), (3, 33, 32), (16, 65536, 20), (1300, 313, 5), (70, 3001, 3), (2, 131073, 32)]:
            logprobs_check(*logits_of(n, V, dtype), top=top)
    monkeypatch.setenv("FRNN_GUARD", "0")
    monkeypatch.setenv("FRNN_CHECK", "1")
    w = rand(11, 16)
    with pytest.raises(runtime.FrnnError, match="outside the vocabulary"):
        fr.embedding(torch.tensor([3, 11], device="cuda"), w)
    assert torch.equal(fr.embedding(torch.tensor([3], device="cuda"), w)[0], w[3])


@pytest.mark.gpu
def test_inputs_without_gradients():
    f, (x, g, b), (up,) = calls()["layer_norm"]
    want = both(f, [x, g, b], [up])
    for need in ([0], [1], [2], [0, 2], [1, 2]):
        leaves = [v if i in need else v.detach() for i, v in enumerate((x, g, b))]
        got = torch.autograd.grad(f(*leaves), [leaves[i] for i in need], up)
        assert all(torch.equal(a, want[1 + i]) for a, i in zip(got, need))
    (bias_only,) = torch.autograd.grad(fr.layer_norm(x.detach(), None, b), b, up)
    assert torch.equal(bias_only, want[3])
    with torch.no_grad():
        assert not fr.layer_norm(x, g, b).requires_grad and torch.equal(fr.layer_norm(x, g, b), want[0])


# ---- what is refused ---------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
def test_refusals():
    t, w, x = torch.zeros(2, 3, dtype=torch.int64, device="cuda"), rand(5, 8), rand(2, 3, 8)
    p = rand(8)
    for call, why in [
            (lambda: fr.embedding(t.float(), w), "int64 or int32"), (lambda: fr.embedding(t, w.double()), "float32, bfloat16 or float16"),
            (lambda: fr.embedding(t, w[0]), "vocabulary, width"), (lambda: fr.embedding(t.cpu(), w), "one CUDA device"),
            (lambda: fr.layer_norm(x.double()), "float32, bfloat16 or float16"), (lambda: fr.layer_norm(x, p[:7]), "width"),
            (lambda: fr.layer_norm(x, p.bfloat16()), "type of x"), (lambda: fr.layer_norm(x, rand(2, 8)), "heads, width"),
            (lambda: fr.layer_norm(x, p, rand(3, 8)), "one shape"), (lambda: fr.layer_norm(x, p.cpu()), "one CUDA device"),
            (lambda: fr.layer_norm(x.bfloat16(), p, p.bfloat16()), "one shape and type"), (lambda: fr.layer_norm(x[0, 0, 0]), "dimension"),
            (lambda: fr.token_logprobs(x, t[:1]), "shape of logits"), (lambda: fr.token_logprobs(x, t.short()), "int64 or int32"),
            (lambda: fr.token_logprobs(x, t, top=9), "top has to be"), (lambda: fr.token_logprobs(rand(2, 3, 80), t, top=33), "top has to be"),
            (lambda: fr.token_logprobs(x, t, top=-1), "top has to be"), (lambda: fr.token_logprobs(x, t, temperature=0.0), "temperature"),
            (lambda: fr.token_logprobs(x, t, temperature=math.nan), "temperature"), (lambda: fr.token_logprobs(x[..., :0], t), "not empty"),
            (lambda: fr.token_logprobs(x, t.cpu()), "one CUDA device"), (lambda: fr.token_logprobs(x.to(torch.float8_e4m3fn), t), "float32, bfloat16 or float16")]:
        with pytest.raises(RuntimeError, match=why):
            call()
    import torch.autograd.forward_ad as ad
    with ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        fr.layer_norm(ad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match="storage"):
        cut = rand(6, 8)
        cut.untyped_storage().resize_(64)
        fr.layer_norm(cut)


def test_refused_on_the_cpu():
    w, x, t = torch.randn(5, 8), torch.randn(3, 8), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: fr.embedding(t, w), lambda: fr.embedding(t, w.requires_grad_()), lambda: fr.layer_norm(x), lambda: fr.token_logprobs(x, t)):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            call()


def test_c_entries_refuse_bad_arguments():
    """Return codes and messages, before anything reaches a device."""
    L = runtime.lib()
    i64, f32, some = ctypes.c_int64, ctypes.c_float, ctypes.c_void_p(256)
    fw = lambda dtype=0, w=some, rows=4, width=8, tok=some, tb=8, n=2, out=some, err=some: L.frnn_embedding_forward(
        dtype, w, i64(rows), i64(width), i64(8), i64(1), tok, tb, i64(n), f32(1), i64(-100), out, err, None)
    assert fw(dtype=7) == fw(tb=2) == fw(w=None) == fw(tok=None) == fw(out=None) == fw(err=None) == fw(rows=1 << 31) == fw(n=-1) == fw(width=-1) == fw(n=1 << 30) == 1
    assert fw(n=0) == fw(width=0) == 0
    bw = lambda dtype=1, dy=some, tok=some, n=2, rows=4, width=8, dw=some, work=some: L.frnn_embedding_backward(
        dtype, dy, tok, 8, i64(n), i64(rows), i64(width), f32(1), i64(-100), dw, work, None)
    assert bw(dtype=3) == bw(dy=None) == bw(tok=None) == bw(dw=None) == bw(work=None) == bw(n=1 << 31) == 1
    assert bw(rows=0) == bw(width=0) == 0
    assert b"2^30" in (bw(n=1 << 31), L.frnn_last_error())[1]

    class Rows(ctypes.Structure):
        _fields_ = [("n", i64 * 3), ("width", i64), ("heads", i64), ("x", i64 * 3), ("dy", i64 * 3), ("dx", i64 * 3)]

    rows = lambda n=(1, 1, 4), width=8, heads=1: ctypes.byref(Rows((i64 * 3)(*n), width, heads))
    ln = lambda r=rows(), dtype=1, x=some, pt=0, y=some: L.frnn_layer_norm_forward(r, dtype, x, pt, None, None, f32(1e-5), y, None, None)
    assert ln(r=None) == ln(dtype=9) == ln(pt=2) == ln(x=None) == ln(y=None) == ln(r=rows(heads=3)) == ln(r=rows(heads=0)) == ln(r=rows(n=(1, 1, -1))) == 1
    assert ln(r=rows(n=(1 << 20, 1 << 20, 1))) == ln(r=rows(width=1 << 31)) == 1
    assert ln(r=rows(n=(0, 1, 4))) == ln(r=rows(width=0)) == 0
    lb = lambda r=rows(), dy=some, x=some, st=some, dx=some, dw=some, work=some: L.frnn_layer_norm_backward(r, 1, dy, x, 0, None, st, dx, dw, None, work, None)
    assert lb(dy=None) == lb(x=None) == lb(st=None) == lb(work=None) == 1
    lp = lambda dtype=0, x=some, n=2, V=8, tok=some, tb=4, top=0, T=1.0, out=some, tl=some, err=some: L.frnn_token_logprobs_forward(
        dtype, x, i64(n), i64(V), i64(V), tok, tb, top, f32(T), i64(-100), out, out, tl, some, None, err, None)
    assert lp(dtype=5) == lp(tb=1) == lp(V=0) == lp(top=33) == lp(top=9) == lp(top=-1) == lp(T=0) == lp(T=math.nan) == lp(T=math.inf) == lp(x=None) == lp(tok=None) == 1
    assert lp(out=None) == lp(top=2, tl=None) == lp(err=None) == lp(n=1 << 31) == lp(V=1 << 30) == 1
    assert lp(n=0) == 0
    odd = ctypes.c_void_p(257)                      # no pointer off the boundary of its elements gets as far as a kernel
    assert fw(w=odd) == fw(tok=odd) == fw(out=odd) == fw(err=odd) == bw(dy=odd) == bw(dw=odd) == bw(work=odd) == ln(x=odd) == ln(y=odd) == lb(st=ctypes.c_void_p(260)) == lb(dx=odd) == 1
    assert lp(x=odd, dtype=1) == lp(out=odd) == lp(tok=odd) == lp(top=2, tl=odd) == 1 and b"boundary" in L.frnn_last_error()
    assert L.frnn_token_logprobs_backward(0, some, i64(2), i64(8), i64(8), some, 8, f32(1), i64(-100), None, None, None, some, None) == 1


def test_definitions_agree_with_torch():
    t = torch.tensor([[1, 4, -100], [0, 1, 2]])
    w, x = torch.randn(5, 6, dtype=torch.double), torch.randn(2, 3, 4, 6, dtype=torch.double)
    y = lm.naive_embedding(t, w, 2.0)
    assert torch.equal(y[0, 1], 2 * w[4]) and not y[0, 2].any()
    g, b = torch.randn(6, dtype=torch.double), torch.randn(6, dtype=torch.double)
    assert torch.allclose(lm.naive_layer_norm(x, g, b), torch.nn.functional.layer_norm(x, (6,), g, b))
    z = torch.randn(2, 3, 5, dtype=torch.double)
    r = lm.naive_token_logprobs(z, t, top=2, temperature=0.5)
    d = torch.distributions.Categorical(logits=z / 0.5)
    assert torch.allclose(r.entropy, d.entropy()) and torch.allclose(r.logprob[1], d.log_prob(t.clamp_min(0))[1]) and r.logprob[0, 2] == 0
    assert torch.equal(r.top_token, z.topk(2).indices)
    z.requires_grad_()
    assert torch.autograd.gradcheck(lambda z: lm.naive_token_logprobs(z, t)[:2], z)


def test_shapes_without_a_gpu():
    """What torch.compile sees: shapes and types, forward and backward."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        ops = (lm._operators(), torch.ops.flex_rnn_b200)[1]
        t, w = torch.zeros(2, 3, dtype=torch.int64, device="cuda"), torch.zeros(5, 8, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        y = fr.embedding(t, w)
        assert y.shape == (2, 3, 8) and y.dtype == torch.bfloat16 and y.requires_grad
        assert ops.embedding_backward(torch.zeros_like(y), t, 5, 1.0, -100).shape == w.shape
        x, p = torch.zeros(2, 3, 4, 8, device="cuda", requires_grad=True), torch.zeros(4, 8, device="cuda", requires_grad=True)
        y, stats = ops.layer_norm(x, p, None, 1e-5, False)
        assert y.shape == x.shape and y.requires_grad and stats.shape == (24, 2) and not stats.requires_grad
        gx, gw, gb = ops.layer_norm_backward(y, x, p, None, stats, True, True, False)
        assert gx.shape == x.shape and gw.shape == p.shape and gb.shape == (0,)
        z = torch.zeros(2, 3, 9, device="cuda", dtype=torch.float16, requires_grad=True)
        r = fr.token_logprobs(z, t, top=4)
        assert r.logprob.shape == (2, 3) and r.entropy.requires_grad and r.top_token.shape == (2, 3, 4) and r.top_token.dtype == torch.int64
        g = ops.token_logprobs_backward(r.logprob, None, z, t, torch.zeros(6, 3, device="cuda"), 1.0, -100)
        assert g.shape == z.shape and g.dtype == z.dtype
