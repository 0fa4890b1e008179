"""gated_mlp, linear_logprobs and rotary (flex_rnn_b200.lm) against their definitions in 64 bits.

Tolerances of the matrix products.  Operands are exact: 16-bit numbers, or fp32 as three bf16 numbers whose products below
2^-24 are left out.  Accumulators have 32 bits and truncate: each instruction adds 16 products and may lose a unit of the last
place, 2^-23 of a partial sum, which is at most the sum S of the terms' absolute values; ``lost(k, dtype)`` counts twice
that for each instruction of a chain (its own alignment of 16 products loses as much at most): k / 16 of them in 16 bits, 16 where parts are added
up in registers, and a rounding for each part of 256 values (fp32: in six products; or 24 for each 64 values, of which
those of the small products, 2^-8 of the sum at most, count for nothing, and a rounding for each).  What lies between two products
is rounded to the operands' type (half a unit in the last place, UNIT); how these errors go on through the formulas
is computed next to the exact results, term by term, with absolute values."""
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

import flex_rnn_b200 as fr
from flex_rnn_b200 import lm, runtime

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
FAST = 2.0 ** -20        # exp, erf and division in 32 bits, with what is left of their arguments' rounding


def rand(*shape, seed=0, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape)), dtype=torch.float32)).cuda()


def off_boundary(t):
    """The values of ``t``, contiguous, one element off a 16-byte boundary."""
    return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)


def lost(k, dtype, in_parts=False):
    parts = k / 256 * (6 if dtype == torch.float32 else 1)
    return (2 * 16 + parts + 8) * 2.0 ** -23 if in_parts or dtype == torch.float32 else 2 * (k / 16 + 8) * 2.0 ** -23


def within(got, want, tol):
    """Everywhere within the tolerance and one rounding of the result."""
    assert got.shape == want.shape
    g = got.detach().double()
    assert torch.isfinite(g).all()
    off = (g - want).abs() - tol - UNIT[got.dtype] * want.abs() - TINY[got.dtype]
    assert not off.numel() or float(off.max()) <= 0, f"{int((off > 0).sum())} of {off.numel()} values off, worst by {float(off.max())} over the tolerance"


def near_in_norm(got, want, roundings):
    """Errors of many values are independent: their 2-norm is that of the roundings on the way (each at most UNIT of a value, 0.6 of it
    in the mean over mantissas and errors), beside which the sums' errors are a few 2^-20."""
    if want.numel() >= 1000:
        assert float((got.detach().double() - want).norm()) <= (UNIT[got.dtype] * roundings ** 0.5 + 2.0 ** -17) * float(want.norm())


# ---- the gated feed-forward block ----------------------------------------------------------------------------------------------

BEND = {"silu": (1.1, 0.5), "gelu": (1.13, 0.8), "relu": (1.0, 0.0), "sigmoid": (0.25, 0.1)}      # largest |act'|, |act''|


def mlp_case(n, D, F, O, dtype, seed=0):
    return [rand(n, D, seed=seed).to(dtype), rand(F, D, seed=seed + 1, scale=D ** -0.5).to(dtype), rand(F, D, seed=seed + 2, scale=D ** -0.5).to(dtype),
            rand(O, F, seed=seed + 3, scale=F ** -0.5).to(dtype)], rand(n, O, seed=seed + 4).to(dtype)


def mlp_exact(x, gate, up, down, dy, activation):
    """(y, dx, dgate, dup, ddown) in 64 bits, and for each how far 32-bit sums and the roundings in between may lead."""
    dtype, (n, D), (O, F) = x.dtype, x.shape, down.shape
    u = 0.0 if dtype == torch.float32 else UNIT[dtype]
    tiny = 0.0 if dtype == torch.float32 else TINY[dtype]
    leaves = [t.detach().double().requires_grad_() for t in (x, gate, up, down)]
    y = lm.naive_gated_mlp(*leaves, activation)
    grads = torch.autograd.grad(y, leaves, dy.double())
    x, gate, up, down = (t.detach() for t in leaves)
    dy = dy.double()
    first, second = BEND[activation]
    a, b = x @ gate.T, x @ up.T
    ea, eb = lost(D, dtype) * (x.abs() @ gate.abs().T), lost(D, dtype) * (x.abs() @ up.abs().T)
    af = a.clone().requires_grad_()
    s = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu, "sigmoid": torch.sigmoid}[activation](af)
    (slope,) = torch.autograd.grad(s.sum(), af)
    s = s.detach()
    h = s * b

    def of_h(ea, eb):
        return first * ea * (b.abs() + eb) + s.abs() * eb + FAST * (a.abs() + 1) * b.abs() + u * h.abs() + tiny

    ey = of_h(ea, eb) @ down.abs().T + lost(F, dtype) * (h.abs() @ down.abs().T)
    dh = dy @ down
    edh = lost(O, dtype) * (dy.abs() @ down.abs())
    es = second * ea + FAST * (a.abs() + 1) + (torch.where(a.abs() <= ea, 1.0, 0.0) if activation == "relu" else 0.0)
    db, da = dh * s, dh * b * slope
    edb = edh * s.abs() + (dh.abs() + edh) * (first * ea + FAST * (s.abs() + 1)) + u * db.abs() + tiny
    eda = edh * (b * slope).abs() + (dh.abs() + edh) * (eb * slope.abs() + (b.abs() + eb) * es) + u * da.abs() + tiny
    edx = eda @ gate.abs() + edb @ up.abs() + lost(2 * F, dtype) * (da.abs() @ gate.abs() + db.abs() @ up.abs())
    ew = [e.T @ x.abs() + lost(n, dtype) * (v.abs().T @ x.abs()) for e, v in ((eda, da), (edb, db))]
    edown = dy.abs().T @ of_h(ea, eb) + lost(n, dtype) * (dy.abs().T @ h.abs())
    return [y.detach(), *grads], [ey, edx, *ew, edown]


def mlp_check(tensors, dy, activation="silu"):
    leaves = [t.detach().requires_grad_() for t in tensors]
    y = fr.gated_mlp(*leaves, activation=activation)
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    flat = [tensors[0].reshape(-1, tensors[0].shape[-1]), *tensors[1:]]
    want, tol = mlp_exact(*flat, dy.reshape(-1, dy.shape[-1]), activation)
    assert y.is_contiguous() and y.dtype == tensors[0].dtype and y.shape == dy.shape
    for g, like, w, t, roundings in zip(got, [y, *tensors], want, tol, (2, 2, 2, 2, 2)):
        assert g.shape == like.shape and g.dtype == like.dtype
        within(g.reshape(w.shape), w, t)
        near_in_norm(g.reshape(w.shape), w, roundings)
    with torch.no_grad():
        assert torch.equal(fr.gated_mlp(*tensors, activation=activation), y)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,D,F,O", [(1, 1, 1, 1), (1, 64, 128, 64), (2, 7, 9, 5), (1, 4096, 640, 33), (16, 1024, 1500, 1024), (37, 100, 77, 131), (128, 64, 64, 64), (129, 65, 257, 63), (777, 485, 1291, 485),
                                     (300, 8, 2049, 16), (2100, 33, 31, 40)])
def test_gated_mlp(n, D, F, O, dtype):
    mlp_check(*mlp_case(n, D, F, O, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,D,F", [(1500, 520, 4000), (2049, 1001, 2050), (4096, 256, 3840)])
def test_gated_mlp_of_large_tiles(n, D, F, dtype):
    """Sizes at which pairs of multiprocessors share a tile, whole and cut off at its edges."""
    mlp_check(*mlp_case(n, D, F, D, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("activation", lm.ACTIVATIONS)
def test_gated_mlp_activations(activation, dtype):
    for n, D, F in ((70, 48, 90), (16, 520, 200)):
        (x, *weights), dy = mlp_case(n, D, F, 40, dtype, seed=3)
        mlp_check([4 * x, *weights], dy, activation)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gated_mlp_layouts(dtype):
    (x, gate, up, down), dy = mlp_case(60, 72, 88, 48, dtype, seed=5)
    want = mlp_check([x, gate, up, down], dy)
    wide = rand(60, 3, 72, seed=6).to(dtype)
    weights = rand(88, 2, 72, seed=7, scale=0.1).to(dtype)
    for t, g in (([off_boundary(v) for v in (x, gate, up, down)], dy), ([x, gate.t().contiguous().t(), up, down.t().contiguous().t()], off_boundary(dy)),
                 ([x.view(5, 12, 72), gate, up, down], dy.view(5, 12, 48)), ([x.view(12, 5, 72), gate, up, down], dy.view(12, 5, 48).transpose(0, 1).contiguous().transpose(0, 1)),
                 ([x.t().contiguous().t(), gate, up, down], dy.t().contiguous().t())):
        got = mlp_check(t, g)
        assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want))
    mlp_check([wide[:, 1], gate, up, down], dy)
    mlp_check([wide[:, 1], weights[:, 0], weights[:, 1], down], dy)
    mlp_check([wide[:, 2, 1:], weights[:, 0, 1:], weights[:, 1, 1:], down], dy)
    mlp_check([x, gate[:, :71].repeat(1, 2)[:, 3:75], up, down], dy)
    mlp_check([x[:1].expand(60, 72), gate, up, down], dy[:1].expand(60, 48))
    mlp_check([x[7], gate, up, down], dy[7])


@pytest.mark.gpu
def test_gated_mlp_empty():
    (x, gate, up, down), _ = mlp_case(4, 16, 24, 8, torch.float32)
    leaves = [v.requires_grad_() for v in (x[:0].detach(), gate, up, down)]
    y = fr.gated_mlp(*leaves)
    assert y.shape == (0, 8)
    for g, v in zip(torch.autograd.grad(y.sum(), leaves), leaves):
        assert torch.equal(g, torch.zeros_like(v))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_mlp_not_finite(dtype):
    """NaN and infinities stay in their rows: rows without any have what they have alone."""
    (x, gate, up, down), dy = mlp_case(200, 64, 96, 64, dtype)
    want = [fr.gated_mlp(x, gate, up, down), *torch.autograd.grad(fr.gated_mlp(x.requires_grad_(), gate, up, down), x, dy)]
    bad = x.detach().clone()
    bad[3, 5], bad[77, 1], bad[199, 63] = math.nan, math.inf, -math.inf
    leaf = bad.requires_grad_()
    y = fr.gated_mlp(leaf, gate, up, down)
    got = [y, *torch.autograd.grad(y, leaf, dy)]
    rows = torch.ones(200, dtype=torch.bool, device="cuda")
    rows[[3, 77, 199]] = False
    for a, b in zip(got, want):
        assert torch.equal(a[rows], b[rows]) and a[3].isnan().all() and not torch.isfinite(a[~rows]).any()


@pytest.mark.gpu
def test_gated_mlp_single_gradients():
    (x, gate, up, down), dy = mlp_case(150, 64, 200, 72, torch.bfloat16)
    leaves = [v.requires_grad_() for v in (x, gate, up, down)]
    want = torch.autograd.grad(fr.gated_mlp(*leaves), leaves, dy)
    for need in ([0], [1], [2], [3], [0, 3], [1, 2], [2, 3]):
        some = [v if i in need else v.detach() for i, v in enumerate(leaves)]
        got = torch.autograd.grad(fr.gated_mlp(*some), [some[i] for i in need], dy)
        assert all(torch.equal(g, want[i]) for g, i in zip(got, need))


# ---- log probabilities without logits -------------------------------------------------------------------------------------------

def logprobs_case(n, V, D, dtype, seed=0, scale=2.0):
    t = torch.randint(0, V, (n,), generator=torch.Generator().manual_seed(seed)).cuda()
    return rand(n, D, seed=seed).to(dtype), rand(V, D, seed=seed + 1, scale=scale * D ** -0.5).to(dtype), t, [rand(n, seed=seed + 2), 0.1 * rand(n, seed=seed + 3)]


def logprobs_exact(x, w, t, up, temperature, ignore):
    """(logprob, entropy, dx, dweight) in 64 bits, and for each how far 32-bit sums and the rounding of the logits' gradient may lead."""
    dtype, (n, D), V = x.dtype, x.shape, w.shape[0]
    leaves = [v.detach().double().requires_grad_() for v in (x, w)]
    r = lm.naive_linear_logprobs(*leaves, t, temperature, ignore)
    grads = torch.autograd.grad(r, leaves, [u.double() for u in up])
    x, w = (v.detach() for v in leaves)
    z = x @ w.T / temperature
    ez = ((lost(D, dtype, True) + 2.0 ** -22) * (x.abs() @ w.abs().T) / temperature).amax(-1)       # of any logit of the row
    again = ((lost(D, dtype) + 2.0 ** -22) * (x.abs() @ w.abs().T) / temperature).amax(-1)           # where the backward computes it again
    logp = torch.log_softmax(z, -1)
    p = logp.exp()
    H = r.entropy.detach()
    size = 1 + math.log(V) + z.abs().amax(-1)
    elp = 2 * ez + 64 * 2.0 ** -24 * size
    eH = 4 * ez * (p * (logp + H[:, None]).abs()).sum(-1) + 4 * ez ** 2 + 64 * 2.0 ** -24 * size
    there = (t != ignore)[:, None]
    g, h = torch.where(there, up[0].double()[:, None], 0.0), up[1].double()[:, None]
    bend = (logp + H[:, None]).abs()
    G = -p * (g + h * (logp + H[:, None]))
    G.scatter_add_(1, torch.where(there, t[:, None], 0), g)
    G /= temperature
    ep = (ez + again + elp + FAST * size)[:, None]                                        # relative error of p
    eG = (p * (g.abs() + h.abs() * bend) * ep * 2 + h.abs() * p * (ep + eH[:, None])) / temperature
    eG = eG + 2.0 ** -22 * (g.abs() + h.abs() * (bend + 1)) / temperature * p + 2.0 ** -23 * G.abs()
    if dtype != torch.float32:
        eG = eG + UNIT[dtype] * G.abs() + 2.0 ** -36 * float((up[0].abs() + 23 * up[1].abs()).max()) / temperature
    edx = eG @ w.abs() + lost(V, dtype) * (G.abs() @ w.abs())
    edw = eG.T @ x.abs() + lost(n, dtype) * (G.abs().T @ x.abs())
    return [r.logprob.detach(), H, *grads], [torch.where(there[:, 0], elp, 0.0), eH, edx, edw]


def logprobs_check(x, w, t, up, temperature=1.0, ignore=-100):
    leaves = [v.detach().requires_grad_() for v in (x, w)]
    r = fr.linear_logprobs(*leaves, t, temperature=temperature, ignore_index=ignore)
    got = [*r, *torch.autograd.grad(r, leaves, up)]
    assert r.logprob.dtype == r.entropy.dtype == torch.float32 and r.logprob.shape == t.shape and got[2].shape == x.shape and got[3].shape == w.shape and got[2].dtype == x.dtype
    want, tol = logprobs_exact(x.reshape(-1, x.shape[-1]), w, t.reshape(-1).long(), [u.reshape(-1) for u in up], temperature, ignore)
    for g, e, tl in zip(got, want, tol):
        within(g.reshape(e.shape), e, tl)
    for g, e in zip(got[2:], want[2:]):
        near_in_norm(g.reshape(e.shape), e, 3)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(fr.linear_logprobs(x, w, t, temperature=temperature, ignore_index=ignore), r))
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (1, 2, 3), (3, 5, 7), (1, 9000, 512), (16, 5003, 1024), (7, 130, 64), (128, 128, 64), (130, 777, 200), (300, 1000, 77), (1030, 257, 24), (500, 3001, 485)])
def test_linear_logprobs(n, V, D, dtype):
    logprobs_check(*logprobs_case(n, V, D, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,D", [(2000, 9001, 256), (1500, 4100, 1001), (4200, 5000, 72)])
def test_linear_logprobs_of_large_tiles(n, V, D, dtype):
    logprobs_check(*logprobs_case(n, V, D, dtype))


@pytest.mark.gpu
def test_linear_logprobs_in_pieces():
    """More rows than a piece of the logits' gradient has room for all of the vocabulary: 2^28 elements, 2^27 in fp32."""
    for n, V, dtype in ((40000, 7001, torch.bfloat16), (30000, 5000, torch.float32), (270000, 1100, torch.float16)):
        x, w, t, up = logprobs_case(n, V, 40, dtype)
        leaves = [x.requires_grad_(), w.requires_grad_()]
        got = torch.autograd.grad(fr.linear_logprobs(*leaves, t), leaves, up)
        total, far = 0.0, 0.0                # the weight's gradient: exact parts of rows, whose chains are all in one sum
        for lo in range(0, n, 5000):
            s = slice(lo, lo + 5000)
            e, tol = logprobs_exact(x.detach()[s], w.detach(), t[s], [u[s] for u in up], 1.0, -100)
            within(got[0][s], e[2], tol[2])
            total, far = total + e[3], far + tol[3]
        within(got[1], total, far * (n / 5000 + 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature", [0.3, 1.7, 25.0])
def test_linear_logprobs_temperature(temperature, dtype):
    logprobs_check(*logprobs_case(90, 500, 64, dtype, seed=4), temperature=temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_logprobs_padding(dtype):
    x, w, t, up = logprobs_case(150, 700, 64, dtype, seed=6)
    t[::3] = -100
    logprobs_check(x, w, t, up)
    logprobs_check(x, w, t.int(), up)
    logprobs_check(x, w, torch.full_like(t, -100), up)
    t[::3] = 5
    logprobs_check(x, w, t, up, ignore=5)
    logprobs_check(x.view(3, 50, 64), w, t.view(3, 50), [u.view(3, 50) for u in up])
    logprobs_check(x[4], w, t[4], [u[4] for u in up])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_logprobs_layouts(dtype):
    x, w, t, up = logprobs_case(60, 300, 72, dtype, seed=8)
    want = logprobs_check(x, w, t, up)
    for a, b, c in ((off_boundary(x), off_boundary(w), t), (x.t().contiguous().t(), w.t().contiguous().t(), torch.stack([t, t], 1)[:, 0]), (x, w, t.int())):
        got = logprobs_check(a, b, c, [off_boundary(u) for u in up])
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    logprobs_check(rand(60, 3, 72, seed=9).to(dtype)[:, 1], rand(300, 80, seed=9, scale=0.2).to(dtype)[:, 5:77], t, up)
    logprobs_check(x[:1].expand(60, 72), w, t, [up[0][:1].expand(60), up[1]])


@pytest.mark.gpu
def test_linear_logprobs_small_gradients_in_fp16():
    """Upstream gradients of a mean over many tokens: most of the logits' gradient lies below fp16's normal numbers.  The gradients
    themselves are scaled up by a power of two (exactly) to be looked at."""
    x, w, t, up = logprobs_case(400, 3000, 64, torch.float16, seed=2)
    for scale in (2.0 ** -14, 2.0 ** -3, 2.0 ** 9):
        leaves = [v.detach().requires_grad_() for v in (x, w)]
        small = [u * scale for u in up]
        r = fr.linear_logprobs(*leaves, t)
        got = torch.autograd.grad(r, leaves, small)
        want, tol = logprobs_exact(x, w, t, small, 1.0, -100)
        within(got[0], want[2], tol[2])
        within(got[1], want[3], tol[3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_logprobs_not_finite(dtype):
    """A row with NaN or an infinity has NaN; the others have what they have alone.  Rows whose logits are all -inf are empty."""
    x, w, t, up = logprobs_case(140, 300, 64, dtype)
    want = logprobs_check(x, w, t, up)
    bad = x.clone()
    bad[3, 5], bad[77, 1] = math.nan, math.inf
    leaf = bad.requires_grad_()
    r = fr.linear_logprobs(leaf, w, t)
    (dx,) = torch.autograd.grad(r, leaf, up)
    rows = torch.ones(140, dtype=torch.bool, device="cuda")
    rows[[3, 77]] = False
    for a, b in zip((*r, dx), want):
        assert torch.equal(a[rows], b[rows]) and a[~rows].isnan().all()
    low = torch.zeros_like(x)
    low[:, 0] = -math.inf if dtype != torch.float32 else 0
    if dtype != torch.float32:          # (an infinity in fp32 meets zeros in the parts of the other operand)
        ones = torch.ones_like(w)
        leaves = [low.requires_grad_(), ones.requires_grad_()]
        r = fr.linear_logprobs(*leaves, t)
        assert (r.logprob == -math.inf).all() and (r.entropy == 0).all()
        dx, dw = torch.autograd.grad(r, leaves, up)
        assert (dx == 0).all()


@pytest.mark.gpu
def test_linear_logprobs_single_outputs():
    x, w, t, up = logprobs_case(100, 300, 48, torch.bfloat16)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    zero = torch.zeros_like(up[0])
    for k in range(2):
        got = torch.autograd.grad(fr.linear_logprobs(*leaves, t)[k], leaves, up[k])
        want = torch.autograd.grad(fr.linear_logprobs(*leaves, t), leaves, [up[k], zero] if k == 0 else [zero, up[k]])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    want = torch.autograd.grad(fr.linear_logprobs(*leaves, t), leaves, up)
    assert torch.equal(torch.autograd.grad(fr.linear_logprobs(x, w.detach(), t), x, up)[0], want[0])
    assert torch.equal(torch.autograd.grad(fr.linear_logprobs(x.detach(), w, t), w, up)[0], want[1])


@pytest.mark.gpu
def test_linear_logprobs_empty():
    x, w, t, _ = logprobs_case(4, 9, 16, torch.float32)
    leaves = [x[:0].detach().requires_grad_(), w.requires_grad_()]
    r = fr.linear_logprobs(*leaves, t[:0])
    assert r.logprob.shape == r.entropy.shape == (0,)
    dx, dw = torch.autograd.grad(r.logprob.sum(), leaves)
    assert dx.shape == (0, 16) and torch.equal(dw, torch.zeros_like(w))


@pytest.mark.gpu
def test_linear_logprobs_token_outside_the_vocabulary():
    x, w, t, _ = logprobs_case(6, 9, 16, torch.bfloat16)
    for bad in (9, -1, 2 ** 31 + 1, -2 ** 40):
        u = t.clone()
        u[2] = bad
        want, got = fr.linear_logprobs(x, w, t), fr.linear_logprobs(x, w, u)
        torch.cuda.synchronize()
        assert got.logprob[2].isnan() and torch.equal(got.entropy, want.entropy) and torch.equal(got.logprob[3:], want.logprob[3:])
        with pytest.raises(runtime.FrnnError, match="outside the vocabulary"):
            fr.linear_logprobs(x, w, t)
        assert torch.equal(fr.linear_logprobs(x, w, t).logprob, want.logprob)


@pytest.mark.gpu
def test_linear_logprobs_equals_token_logprobs():
    """The same results as from logits, to the precision of fp32 products."""
    x, w, t, up = logprobs_case(64, 1000, 96, torch.float32)
    got = logprobs_check(x, w, t, up)
    other = fr.token_logprobs((x.double() @ w.double().T).float(), t)
    size = (x.double().abs() @ w.double().abs().T).amax(-1)
    for a, b in zip(got[:2], other[:2]):
        assert ((a - b).abs().double() <= 8 * lost(96, torch.float32) * size * (1 + math.log(1000))).all()


# ---- rotary positions -------------------------------------------------------------------------------------------------------------

def rotary_check(x, positions, frequencies, interleaved=False, scale=1.0, seed=1):
    leaf = x.detach().requires_grad_()
    y = fr.rotary(leaf, positions, frequencies, interleaved=interleaved, scale=scale)
    dy = rand(*x.shape, seed=seed).to(x.dtype)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    exact = x.detach().double().requires_grad_()
    want = lm.naive_rotary(exact, positions, frequencies.double(), interleaved, scale)
    (dwant,) = torch.autograd.grad(want, exact, dy.double())
    pairs = 2 * frequencies.shape[0]
    assert y.is_contiguous() and y.dtype == x.dtype
    for got, w, v in ((y, want.detach(), x), (dx, dwant, dy)):
        # |u cos| + |w sin| is at most the pair's norm times sqrt 2; sine, cosine, the angle's rest, two products and a sum: 2^-24 of it each, twice over
        v = v.detach().double()
        a, b = (v[..., 0:pairs:2], v[..., 1:pairs:2]) if interleaved else (v[..., :pairs // 2], v[..., pairs // 2:pairs])
        size = torch.hypot(a, b) * scale * 1.5
        size = torch.stack([size, size], -1).flatten(-2) if interleaved else torch.cat([size, size], -1)
        within(got[..., :pairs], w[..., :pairs], 12 * 2.0 ** -24 * size)
        assert torch.equal(got[..., pairs:], v[..., pairs:].to(x.dtype))
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,H,N,pairs", [(1, 1, 1, 2, 1), (2, 3, 4, 64, 32), (1, 7, 3, 97, 31), (16, 1, 64, 128, 64), (2, 5, 1, 20, 10), (1, 300, 2, 96, 20), (3, 11, 5, 36, 18), (1, 2, 7, 256, 128), (1, 3, 2, 1100, 530),
                                           (2, 1, 33, 24, 4), (1, 1, 1, 7, 0), (5, 1000, 3, 16, 8)])
def test_rotary(B, T, H, N, pairs, interleaved, dtype):
    x = rand(B, T, H, N).to(dtype)
    f = lm.rotary_frequencies(2 * pairs, device="cuda")
    rotary_check(x, 0, f, interleaved)
    rotary_check(x, torch.randint(-50, 2 ** 21, (B, T), generator=torch.Generator().manual_seed(3)).cuda(), f, interleaved, scale=1.3)


@pytest.mark.gpu
def test_rotary_layouts():
    f = lm.rotary_frequencies(32, base=500.0, device="cuda")
    p = (torch.arange(10, device="cuda") * 7 + torch.tensor([[3], [100000], [5]], device="cuda"))
    for dtype in (torch.float32, torch.bfloat16):
        for x in (rand(3, 10, 4, 40).to(dtype), rand(3, 4, 10, 40).to(dtype).transpose(1, 2), rand(3, 10, 12, 40).to(dtype)[:, :, 4:8], rand(3, 10, 4, 1, 40).to(dtype), rand(3, 10, 40).to(dtype), rand(3, 10, 2, 3, 40).to(dtype),
                  rand(3, 10, 3, 2, 40).to(dtype).transpose(2, 3), rand(3, 10, 4, 45).to(dtype)[..., 3:43], off_boundary(rand(3, 10, 4, 40).to(dtype)), rand(10, 3, 4, 40).to(dtype).transpose(0, 1),
                  rand(3, 10, 40, 4).to(dtype).transpose(2, 3), rand(1, 10, 1, 40).to(dtype).expand(3, 10, 4, 40)):
            for interleaved in (False, True):
                for where in (p, p.int(), p[1], p[:1], p.t().contiguous().t(), 12345, torch.stack([p, p], -1)[..., 0]):
                    rotary_check(x, where, f, interleaved, scale=0.7)
                rotary_check(x, p, f.float(), interleaved)
                rotary_check(x, p, torch.stack([f, f], 1)[:, 0], interleaved)


@pytest.mark.gpu
def test_rotary_far_positions():
    """A turn's rest does not depend on how many turns lie before it."""
    x = rand(1, 6, 2, 64)
    rotary_check(x, torch.tensor([2 ** 20 - 1, 10 ** 7, -10 ** 7, 2 ** 31 + 5, -1, 0], device="cuda"), lm.rotary_frequencies(64, device="cuda"))


@pytest.mark.gpu
def test_rotary_offsets_past_31_bits():
    x = torch.zeros(1, 70000, 4, 8200, dtype=torch.bfloat16, device="cuda")      # 2.3 10^9 elements
    x[0, -1] = rand(4, 8200)
    f = lm.rotary_frequencies(128, device="cuda")
    y = fr.rotary(x, 7, f)
    want = fr.rotary(x[:, -1:].clone(), 7 + 69999, f)
    assert torch.equal(y[:, -1:], want) and not y[:, :-1].any()


@pytest.mark.gpu
def test_rotary_empty_and_twice_differentiable():
    f = lm.rotary_frequencies(8, device="cuda")
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        y = fr.rotary(x, 0, f)
        assert y.shape == shape and torch.autograd.grad(y.sum(), x)[0].shape == shape
    x, dy = rand(2, 3, 4, 8).requires_grad_(), rand(2, 3, 4, 8, seed=2).requires_grad_()
    (dx,) = torch.autograd.grad(fr.rotary(x, 5, f, scale=2.0), x, dy, create_graph=True)
    (back,) = torch.autograd.grad(dx, dy, x.detach())
    assert torch.equal(back, fr.rotary(x.detach(), 5, f, scale=2.0))


def test_rotary_frequencies():
    f = lm.rotary_frequencies(64, base=100.0)
    assert f.dtype == torch.float64 and f.shape == (32,) and f[0] == 1
    torch.testing.assert_close(f, torch.tensor([100.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64), rtol=1e-14, atol=0)
    assert torch.equal(lm.rotary_frequencies(64, base=100.0, factor=8.0), f / 8)
    g = lm.rotary_frequencies(64, base=100.0, factor=8.0, method="base")
    assert g[0] == 1
    torch.testing.assert_close(g[-1], f[-1] / 8, rtol=1e-14, atol=0)
    g = lm.rotary_frequencies(64, base=10000.0, factor=8.0, method="parts", length=2048)
    f = lm.rotary_frequencies(64, base=10000.0)
    turns = 2048 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.equal(g[turns <= 1], f[turns <= 1] / 8) and (g.diff() < 0).all() and ((g <= f) & (g >= f / 8)).all()
    assert lm.rotary_frequencies(0).shape == (0,) and torch.equal(lm.rotary_frequencies(2, method="base", factor=3.0), torch.ones(1, dtype=torch.float64))
    for bad in (dict(width=3), dict(width=-2), dict(width=4, base=0.0), dict(width=4, factor=-1.0), dict(width=4, method="other"), dict(width=4, method="parts"), dict(width=4, method="parts", length=9, turns=(3, 2))):
        with pytest.raises(ValueError):
            lm.rotary_frequencies(**bad)


# ---- all of them ------------------------------------------------------------------------------------------------------------------

NAMES = ["gated_mlp", "linear_logprobs", "rotary"]


def calls(dtype=torch.float32, device="cuda"):
    """name -> (function of its leaves, the leaves, upstream gradients)"""
    r = (lambda *s, **k: rand(*s, **k).to(device)) if device == "cuda" else (lambda *s, **k: torch.empty(*s, device=device))
    t = (torch.arange(60, device=device) * 7 % 50).view(3, 20)
    p, f = torch.arange(20, device=device) + 9, lm.rotary_frequencies(32, device=device)
    one = lambda f: lambda *a: (f(*a),)
    out = {"gated_mlp": (one(fr.gated_mlp), [r(3, 20, 48), r(72, 48, seed=1, scale=0.15), r(72, 48, seed=2, scale=0.15), r(40, 72, seed=3, scale=0.1)], [r(3, 20, 40, seed=6)]),
           "linear_logprobs": (lambda x, w: tuple(fr.linear_logprobs(x, w, t, temperature=0.9)), [r(3, 20, 48), r(50, 48, seed=1, scale=0.3)], [r(3, 20, seed=7), r(3, 20, seed=8)]),
           "rotary": (one(lambda x: fr.rotary(x, p, f, scale=1.5)), [r(3, 20, 4, 40)], [r(3, 20, 4, 40, seed=9)])}
    return {k: (f, [v.to(dtype).requires_grad_() for v in a], [u if k == "linear_logprobs" else u.to(dtype) for u in up]) for k, (f, a, up) in out.items()}


def both(f, leaves, up):
    y = f(*leaves)
    return [*(v.detach() for v in y), *torch.autograd.grad(y, leaves, up)]


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_gradients_against_differences(name):
    """Central differences of the operator's own forward along random directions, in fp32.  Truncation: the third
    derivative along d is at most about 30 (values of order 1), times h^2 / 6; rounding: 2^-20 of each output, in random
    directions, over 2 h."""
    f, leaves, up = calls()[name]
    grads = torch.autograd.grad(f(*leaves), leaves, up)
    h = 2.0 ** -6
    value = lambda a: [y.double() for y in f(*a)]
    for i, (leaf, g) in enumerate(zip(leaves, grads)):
        for seed in range(3):
            d = rand(*leaf.shape, seed=40 + seed)
            d = d / d.norm() * 4
            step = lambda s: [v.detach() + (s * d if j == i else 0) for j, v in enumerate(leaves)]
            hi, lo = value(step(h)), value(step(-h))
            diff = sum(float(((a - b) * u.double()).sum()) for a, b, u in zip(hi, lo, up)) / (2 * h)
            size = sum(float(u.double().norm() * a.norm()) for a, u in zip(hi, up))
            bend = 30 * float(d.abs().max()) ** 2 * sum(float(u.double().norm()) for u in up) * 4
            assert abs(diff - float((g.double() * d.double()).sum())) <= 2.0 ** -20 * size / (2 * h) + bend * h * h / 6


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_repeated_calls_give_the_same_bits(name):
    f, leaves, up = calls(torch.bfloat16)[name]
    want = both(f, leaves, up)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(both(f, leaves, up), want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_streams_and_graphs(name):
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
    for _ in range(2):
        with torch.no_grad():
            for a, b in zip(still, leaves):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_threads(name):
    """Calls from several threads, each on a stream of its own and at once, give what one thread gives."""
    import threading
    f, leaves, up = calls()[name]
    want = both(f, leaves, up)
    torch.cuda.synchronize()
    wrong = []

    def work():
        try:
            mine, side = [v.detach().clone().requires_grad_() for v in leaves], torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for _ in range(20):
                    got = both(f, mine, up)
                    side.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want)):
                        wrong.append("other results")
        except Exception as e:
            wrong.append(repr(e))

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_compiled(name):
    f, leaves, up = calls()[name]
    plain = lambda *a: tuple(2 * v for v in f(*a))
    compiled = torch.compile(plain, fullgraph=True, dynamic=False)
    for a, b in zip(both(compiled, leaves, up), both(plain, leaves, up)):
        assert a.dtype == b.dtype and torch.equal(a, b)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(compiled(*leaves), plain(*leaves)))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_graph_semantics(name):
    """Second use, changed inputs, saved-tensor hooks, batched upstream gradients, gradients of gradients."""
    f, leaves, up = calls()[name]
    want = both(f, leaves, up)[-len(leaves):]
    if name != "rotary":
        for wrt in (0, -1):
            ups = [u.detach().requires_grad_() for u in up]
            first = torch.autograd.grad(f(*leaves), leaves, ups, create_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(first, want))
            with pytest.raises(RuntimeError, match="not differentiable"):
                torch.autograd.grad(first[wrt].sum(), [leaves[0], ups[0]])
    y = f(*leaves)
    torch.autograd.grad(y, leaves, up)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, leaves, up)
    hooks = torch.autograd.graph.saved_tensors_hooks
    for ctx in (torch.autograd.graph.save_on_cpu(pin_memory=True), hooks(off_boundary, lambda t: t), hooks(lambda t: t.t().contiguous() if t.dim() == 2 else t, lambda t: t.t() if t.dim() == 2 else t)):
        with ctx:
            y = f(*leaves)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, up), want))
    many = torch.autograd.grad(f(*leaves), leaves, [torch.stack([u, -2 * u]) for u in up], is_grads_batched=True)
    for a, b in zip(many, want):
        assert torch.equal(a[0], b) and torch.equal(a[1], -2 * b)
    if name != "rotary":
        y = f(*leaves)
        with torch.no_grad():
            leaves[0].add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, leaves, up)


@pytest.mark.gpu
def test_guard_bands(monkeypatch):
    """With FRNN_GUARD=1 no kernel writes outside of its buffers."""
    monkeypatch.setenv("FRNN_GUARD", "1")
    for dtype in DTYPES:
        for n, D, F, O in [(1, 1, 1, 1), (16, 1024, 1500, 1024), (129, 65, 257, 63), (1500, 520, 4000, 520)]:
            mlp_check(*mlp_case(n, D, F, O, dtype))
        for n, V, D in [(1, 2, 3), (16, 5003, 1024), (130, 777, 200), (2000, 9001, 256)]:
            logprobs_check(*logprobs_case(n, V, D, dtype))
        for B, T, H, N, pairs in [(1, 1, 1, 2, 1), (2, 3, 4, 64, 32), (1, 7, 3, 97, 31)]:
            rotary_check(rand(B, T, H, N).to(dtype), 3, lm.rotary_frequencies(2 * pairs, device="cuda"), True)


@pytest.mark.gpu
def test_first_use_is_a_captured_one():
    """A process whose first use of each operator, forward and backward, is captured into a graph."""
    program = """
import torch, flex_rnn_b200 as fr
g = torch.Generator(device="cuda").manual_seed(0)
r = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16().requires_grad_()
x, gate, up, down, w, t = r(300, 96), r(200, 96), r(200, 96), r(96, 200), r(1000, 96), torch.arange(300, device="cuda")
f = fr.rotary_frequencies(96, device="cuda")
def step():
    y = fr.gated_mlp(fr.rotary(x.view(1, 300, 1, 96), 5, f).view(300, 96), gate, up, down)
    lp = fr.linear_logprobs(y, w, t).logprob
    return [lp, *torch.autograd.grad(lp.sum(), [x, gate, up, down, w])]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
print(all(torch.equal(a, b) for a, b in zip(got, step())))
"""
    r = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), timeout=600)
    assert r.stdout.split() == ["True"], r.stdout + r.stderr[-2000:]


# ---- what is refused ----------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
def test_refusals():
    x, g, d, t, f = rand(2, 3, 8), rand(12, 8), rand(5, 12), torch.zeros(2, 3, dtype=torch.int64, device="cuda"), lm.rotary_frequencies(8, device="cuda")
    q = x[:, :, None]
    for call, why in [
            (lambda: fr.gated_mlp(x.double(), g, g, d), "float32, bfloat16 or float16"), (lambda: fr.gated_mlp(x, g.bfloat16(), g, d), "type of x"), (lambda: fr.gated_mlp(x, g[:, :7], g[:, :7], d), "hidden, width"),
            (lambda: fr.gated_mlp(x, g, g[:11], d), "hidden, width"), (lambda: fr.gated_mlp(x, g, g, d[:, :11]), "out, hidden"), (lambda: fr.gated_mlp(x, g[0], g, d), "matrix"), (lambda: fr.gated_mlp(x, g.cpu(), g, d), "one CUDA device"),
            (lambda: fr.gated_mlp(x[..., :0], g[:, :0], g[:, :0], d), "width that is not 0"), (lambda: fr.gated_mlp(x, g[:0], g[:0], d[:, :0]), "not empty"), (lambda: fr.gated_mlp(x[0, 0, 0], g, g, d), "width"),
            (lambda: fr.linear_logprobs(x.double(), g, t), "float32, bfloat16 or float16"), (lambda: fr.linear_logprobs(x, g.half(), t), "type of x"), (lambda: fr.linear_logprobs(x, g[:, :7], t), "vocabulary, width"),
            (lambda: fr.linear_logprobs(x, g, t[:1]), "shape of x"), (lambda: fr.linear_logprobs(x, g, t.short()), "int64 or int32"), (lambda: fr.linear_logprobs(x, g, t, temperature=0.0), "temperature"),
            (lambda: fr.linear_logprobs(x, g, t, temperature=math.nan), "temperature"), (lambda: fr.linear_logprobs(x, g[:0], t), "not empty"), (lambda: fr.linear_logprobs(x, g, t.cpu()), "one CUDA device"),
            (lambda: fr.rotary(x[0], 0, f), "batch, length"), (lambda: fr.rotary(q.double(), 0, f), "float32, bfloat16 or float16"), (lambda: fr.rotary(q, 0, lm.rotary_frequencies(10, device="cuda")), "a head has 8"),
            (lambda: fr.rotary(q, 0, f.half()), "float32 or float64"), (lambda: fr.rotary(q, 0, f[None]), "vector"), (lambda: fr.rotary(q, t.float(), f), "int64 or int32"), (lambda: fr.rotary(q, t[:, :2], f), "positions have to be"),
            (lambda: fr.rotary(q, t.new_zeros(3, 3), f), "positions have to be"), (lambda: fr.rotary(q, 0, f.cpu()), "one CUDA device"), (lambda: fr.rotary(q, t.cpu(), f), "one CUDA device"),
            (lambda: fr.rotary(q, 0, f.clone().requires_grad_()), "no gradient")]:
        with pytest.raises(RuntimeError, match=why):
            call()
    import torch.autograd.forward_ad as ad
    for call in (lambda v: fr.gated_mlp(v, g, g, d), lambda v: fr.linear_logprobs(v, g, t), lambda v: fr.rotary(v[:, :, None], 0, f)):
        with ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            call(ad.make_dual(x, torch.ones_like(x)))


def test_refused_on_the_cpu():
    x, w, d, t, f = torch.randn(2, 3, 8), torch.randn(5, 8), torch.randn(8, 5), torch.zeros(2, 3, dtype=torch.int64), lm.rotary_frequencies(8)
    for call in (lambda: fr.gated_mlp(x, w, w, d), lambda: fr.linear_logprobs(x, w.requires_grad_(), t), lambda: fr.rotary(x[:, :, None], 0, f)):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            call()
    with pytest.raises(ValueError, match="activation"):
        fr.gated_mlp(x, w, w, d, activation="tanh")


def test_c_entries_refuse_bad_arguments():
    L, vp, i64, i32 = runtime.lib(), ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32

    class Mlp(ctypes.Structure):
        _fields_ = [("dtype", i32), ("activation", i32), *[(k, i64) for k in ("n", "width", "hidden", "out_width")], *[(k, vp) for k in ("x", "gate", "up", "down")],
                    *[(k, i64) for k in ("x_stride", "gate_stride", "up_stride", "down_stride")]]

    class Logprobs(ctypes.Structure):
        _fields_ = [("dtype", i32), ("token_bytes", i32), *[(k, i64) for k in ("n", "vocab", "width")], ("x", vp), ("weight", vp), ("x_stride", i64), ("weight_stride", i64), ("tokens", vp),
                    ("ignore_index", i64), ("temperature", ctypes.c_float)]

    class Rotary(ctypes.Structure):
        _fields_ = [*[(k, i32) for k in ("dtype", "interleaved", "inverse", "position_bytes", "frequency_bytes")], ("scale", ctypes.c_float), *[(k, i64) for k in ("batch", "length", "heads", "width", "pairs", "start")],
                    ("x_stride", i64 * 3), ("y_stride", i64 * 3), ("position_stride", i64 * 2)]

    P = vp(4096)
    p = 4096
    for f in ("frnn_gated_mlp_forward_workspace", "frnn_gated_mlp_backward_workspace", "frnn_linear_logprobs_forward_workspace", "frnn_linear_logprobs_backward_workspace"):
        getattr(L, f).restype = ctypes.c_size_t
    mlp = dict(dtype=1, activation=0, n=4, width=8, hidden=16, out_width=8, x=p, gate=p, up=p, down=p, x_stride=8, gate_stride=8, up_stride=8, down_stride=16)
    forward = lambda c, y=P, a=None, b=None, h=None, work=P, err=P: L.frnn_gated_mlp_forward(c and ctypes.byref(c), y, a, b, h, work, err, None)
    backward = lambda c, dy=P, stride=8, a=P, b=P, h=P, dx=P, work=P, err=P: L.frnn_gated_mlp_backward(c and ctypes.byref(c), dy, i64(stride), a, b, h, dx, None, None, None, work, err, None)
    assert L.frnn_gated_mlp_forward_workspace(ctypes.byref(Mlp(**mlp))) > 0 and L.frnn_gated_mlp_backward_workspace(ctypes.byref(Mlp(**mlp)), P, i64(8)) > 0
    for bad in (dict(dtype=3), dict(dtype=-1), dict(activation=4), dict(activation=-1), dict(n=0), dict(n=2 ** 31), dict(width=0), dict(hidden=-1), dict(out_width=2 ** 31), dict(x=None), dict(gate=p + 1), dict(down=p + 1),
                dict(x_stride=-8), dict(up_stride=2 ** 40)):
        c = Mlp(**{**mlp, **bad})
        assert forward(c) == 1 and backward(c) == 1 and L.frnn_gated_mlp_forward_workspace(ctypes.byref(c)) == 0 and L.frnn_gated_mlp_backward_workspace(ctypes.byref(c), P, i64(8)) == 0
    c = Mlp(**mlp)
    for rc in (forward(None), forward(c, y=None), forward(c, y=vp(p + 1)), forward(c, a=P), forward(c, b=P), forward(c, a=P, b=P), forward(c, h=P), forward(c, a=vp(p + 2), b=P, h=P), forward(c, a=P, b=P, h=vp(p + 8)), forward(c, work=None), forward(c, work=vp(p + 8)), forward(c, err=None),
               backward(None), backward(c, dy=None), backward(c, dy=vp(p + 1)), backward(c, stride=-1), backward(c, a=None), backward(c, b=vp(p + 4)), backward(c, h=None), backward(c, h=vp(p + 2)), backward(c, dx=vp(p + 1)), backward(c, work=None), backward(c, err=None)):
        assert rc == 1
    assert backward(c, dx=None) == 0                      # (nothing is wanted)

    lp = dict(dtype=1, token_bytes=8, n=4, vocab=100, width=8, x=p, weight=p, x_stride=8, weight_stride=8, tokens=p, ignore_index=-100, temperature=1.0)
    forward = lambda c, lp=P, ent=P, stats=None, work=P, err=P: L.frnn_linear_logprobs_forward(c and ctypes.byref(c), lp, ent, stats, work, err, None)
    backward = lambda c, g=P, h=P, stats=P, dx=P, dw=P, work=P, err=P: L.frnn_linear_logprobs_backward(c and ctypes.byref(c), g, h, stats, dx, dw, work, err, None)
    assert L.frnn_linear_logprobs_forward_workspace(ctypes.byref(Logprobs(**lp))) > 0 and L.frnn_linear_logprobs_backward_workspace(ctypes.byref(Logprobs(**lp))) > 0
    for bad in (dict(dtype=7), dict(token_bytes=2), dict(n=0), dict(n=2 ** 30), dict(vocab=0), dict(vocab=2 ** 30), dict(width=0), dict(x=None), dict(weight=None), dict(tokens=None), dict(tokens=p + 4), dict(x=p + 1), dict(weight=p + 1),
                dict(x_stride=-1), dict(weight_stride=2 ** 40), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf)):
        c = Logprobs(**{**lp, **bad})
        assert forward(c) == 1 and backward(c) == 1 and L.frnn_linear_logprobs_forward_workspace(ctypes.byref(c)) == 0 and L.frnn_linear_logprobs_backward_workspace(ctypes.byref(c)) == 0
    c = Logprobs(**lp)
    for rc in (forward(None), forward(c, lp=None), forward(c, ent=None), forward(c, lp=vp(p + 2)), forward(c, stats=vp(p + 2)), forward(c, work=None), forward(c, work=vp(p + 4)), forward(c, err=None), backward(None), backward(c, stats=None),
               backward(c, g=vp(p + 2)), backward(c, h=vp(p + 1)), backward(c, dx=vp(p + 1)), backward(c, dw=vp(p + 1)), backward(c, work=None), backward(c, err=None)):
        assert rc == 1
    assert backward(c, dx=None, dw=None) == 0

    rot = dict(dtype=1, interleaved=0, inverse=0, position_bytes=8, frequency_bytes=8, scale=1.0, batch=1, length=2, heads=3, width=8, pairs=4, start=0)
    call = lambda x=P, where=P, f=P, y=P, **bad: L.frnn_rotary(ctypes.byref(Rotary(**{**rot, **bad})), x, where, f, y, None)
    for rc in (L.frnn_rotary(None, P, P, P, P, None), call(dtype=5), call(position_bytes=2), call(frequency_bytes=2), call(batch=-1), call(length=2 ** 31), call(heads=-1), call(pairs=5), call(pairs=-1), call(width=-1), call(x=None), call(y=None),
               call(f=None), call(x=vp(p + 1)), call(y=vp(p + 1)), call(where=vp(p + 4)), call(f=vp(p + 4))):
        assert rc == 1
    assert call(batch=0) == 0 and call(heads=0) == 0


def test_definitions_agree_with_torch():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    x, gate, up, down, t = r(3, 5, 8), r(12, 8), r(12, 8), r(7, 12), torch.randint(0, 12, (3, 5), generator=g)
    linear = torch.nn.functional.linear
    torch.testing.assert_close(lm.naive_gated_mlp(x, gate, up, down), linear(torch.nn.functional.silu(linear(x, gate)) * linear(x, up), down))
    q = lm.naive_linear_logprobs(x, gate, t, 0.7)
    torch.testing.assert_close(-q.logprob, torch.nn.functional.cross_entropy(linear(x, gate).view(15, 12) / 0.7, t.view(15), reduction="none").view(3, 5))
    torch.testing.assert_close(q.entropy, torch.distributions.Categorical(logits=linear(x, gate) / 0.7).entropy())
    f = lm.rotary_frequencies(6)
    for interleaved in (False, True):
        y = lm.naive_rotary(x[:, :, None], 3, f, interleaved, 2.0)[:, :, 0]
        pairs = x[..., :6].unflatten(-1, (3, 2)) if interleaved else x[..., :6].unflatten(-1, (2, 3)).transpose(-1, -2)
        z = torch.view_as_real(2.0 * torch.view_as_complex(pairs.contiguous()) * torch.exp(1j * (3 + torch.arange(5).double())[:, None] * f))
        torch.testing.assert_close(y[..., :6], z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2))
        assert torch.equal(y[..., 6:], x[..., 6:])


@pytest.mark.parametrize("name", NAMES)
def test_shapes_without_a_gpu(name):
    """Results and gradients have their shapes on meta tensors, also traced with symbolic sizes; tangents on upstream gradients are
    refused where gradients are not differentiable."""
    import torch.autograd.forward_ad as ad
    lm._operators()
    f, leaves, up = calls(device="meta")[name]
    assert [g.shape for g in torch.autograd.grad(f(*leaves), leaves, up)] == [v.shape for v in leaves]
    assert [y.shape for y in f(*leaves)] == [u.shape for u in up]
    if name != "rotary":
        with ad.dual_level():
            up[0] = ad.make_dual(up[0], torch.empty_like(up[0]))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(f(*leaves), leaves, up)


OF_BATCH = {"gated_mlp": (lambda x, g, d: (fr.gated_mlp(x, g, g, d),), lambda b, e: ([e(b, 7, 24), e(40, 24), e(24, 40)], [e(b, 7, 24)])),
            "linear_logprobs": (lambda x, w: tuple(fr.linear_logprobs(x, w, torch.zeros(x.shape[:2], dtype=torch.int64, device=x.device))), lambda b, e: ([e(b, 7, 24), e(11, 24)], [e(b, 7), e(b, 7)])),
            "rotary": (lambda x, f: (fr.rotary(x, 5, f.detach()) + 0 * f.sum().to(x.dtype),), lambda b, e: ([e(b, 7, 2, 24), e(6)], [e(b, 7, 2, 24)]))}


def of_batch(name, b, device):
    f, make = OF_BATCH[name]
    leaves, up = make(b, lambda *s: torch.linspace(-2, 3, math.prod(s), device=device).sin().view(s))
    return f, [v.requires_grad_() for v in leaves], up


@pytest.mark.parametrize("name", NAMES)
def test_symbolic_sizes(name):
    lm._operators()
    torch._dynamo.reset()
    compiled = torch.compile(lambda f, a: f(*a), fullgraph=True, backend="aot_eager", dynamic=True)
    for b in (6, 7, 9):
        f, leaves, up = of_batch(name, b, "meta")
        assert [g.shape for g in torch.autograd.grad(compiled(f, leaves), leaves, up)] == [v.shape for v in leaves]


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_compiled_for_any_batch(name):
    torch._dynamo.reset()
    compiled = torch.compile(lambda f, a: f(*a), fullgraph=True, dynamic=True)
    for b in (6, 7, 9):
        f, leaves, up = of_batch(name, b, "cuda")
        assert all(torch.equal(a, g) for a, g in zip(both(lambda *a: compiled(f, a), leaves, up), both(f, leaves, up)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("n,V,D", [(1, 300, 64), (9, 3000, 383), (40, 1000, 72), (128, 515, 200)])
def test_gradients_of_few_rows(n, V, D, dtype):
    """Up to 128 rows the logits' gradient G is multiplied in two parts, 2^-16 of it (fp16: 2^-22, but not below its least number): beside the
    result's rounding there are 2^-14 of |G| |W| and |G|^T |x|, in which logits' and sums' errors (2^-17 each) have room."""
    x, w = rand(n, D).to(dtype), rand(V, D, scale=D ** -0.5).to(dtype)
    t, g, h = torch.arange(n).cuda() * 7 % V, rand(n, seed=1), rand(n, seed=2, scale=0.01)
    t[n // 2] = -100
    leaves = [v.requires_grad_() for v in (x, w)]
    exact = [v.detach().double().requires_grad_() for v in leaves]
    r = fr.linear_logprobs(*leaves, t, temperature=0.7)
    got = torch.autograd.grad([r.logprob, r.entropy], leaves, [g, h])
    logits = (exact[0] @ exact[1].t()).detach().requires_grad_()
    s = lm.naive_token_logprobs(logits, t, 0, 0.7)
    G, = torch.autograd.grad([s[0], s[1]], logits, [g.double(), h.double()])
    for a, b, size in ((got[0], G @ exact[1], G.abs() @ exact[1].abs()), (got[1], G.t() @ exact[0], G.abs().t() @ exact[0].abs())):
        within(a, b.detach(), 2.0 ** -14 * size.detach())


def turned_from(device):
    """A compiled rotation of single tokens, as generation calls it, from many positions: two programs, not one for each."""
    lm._operators()
    torch._dynamo.reset()
    f = torch.linspace(1, 0.1, 4, dtype=torch.float64, device=device)
    x = torch.ones(2, 1, 3, 10, device=device, requires_grad=True)
    compiled = torch.compile(lambda x, p: fr.rotary(x, p, f), fullgraph=True, backend="aot_eager")
    for p in [0, 5, 2 ** 40, *range(7, 30)]:
        y = compiled(x, p)
        yield x, y, fr.rotary(x, p, f)


def test_symbolic_position():
    for x, y, want in turned_from("meta"):
        assert y.shape == want.shape and torch.autograd.grad(y.sum(), x)[0].shape == x.shape


@pytest.mark.gpu
def test_compiled_for_any_position():
    for x, y, want in turned_from("cuda"):
        assert torch.equal(y, want) and torch.equal(*(torch.autograd.grad(v.sum(), x)[0] for v in (y, want)))


@pytest.mark.gpu
def test_gelu_everywhere():
    """gelu and its derivative alone, from x = (a, 1), gate (1, 0), up (0, 1), down 1.  Relative errors in units of 2^-24, with t = |a|: the exponent
    t^2 / 2 is rounded three times (1.5 t^2), an exponential 4, a reciprocal 5 (times 1.3, as it goes into the polynomial), the polynomial 4, four
    roundings behind it, products on the way 4: 24 + 1.5 t^2 of each term."""
    a = torch.cat([torch.linspace(-12, 12, 20001), torch.tensor([0.0, -0.0, 1e-30, -1e-30, 30.0, -30.0, 1e30, -1e30])]).cuda()
    x = torch.stack([a, torch.ones_like(a)], -1).requires_grad_()
    gate, up, down = torch.tensor([[1.0, 0.0]]).cuda(), torch.tensor([[0.0, 1.0]]).cuda(), torch.ones(1, 1).cuda()
    y = fr.gated_mlp(x, gate, up, down, "gelu")
    slope = torch.autograd.grad(y.sum(), x)[0][:, 0].double()
    t = a.double()
    share, density = 0.5 * torch.special.erfc(-t / 2 ** 0.5), torch.exp(-t * t / 2) / (2 * math.pi) ** 0.5
    tol = (24 + 1.5 * t * t) * 2.0 ** -24
    for got, terms in ((y[:, 0].double(), (t * share,)), (slope, (share, torch.where(density == 0, 0.0, t * density)))):
        off = (got - sum(terms)).abs() - tol.clamp(max=1.0) * sum(v.abs() for v in terms) - 2.0 ** -120
        assert float(off.max()) <= 0, (float(a[off.argmax()]), float(off.max()))
    inf = fr.gated_mlp(torch.tensor([[math.nan, 1.0]]).cuda(), gate, up, down, "gelu")
    assert inf.isnan().all()
