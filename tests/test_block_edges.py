"""Calls of gated_mlp, linear_logprobs and rotary (flex_rnn_b200.lm) at their edges; tolerances are those of test_block."""
import ctypes
import math

import pytest
import torch

import flex_rnn_b200 as fr
from flex_rnn_b200 import lm, runtime
from flex_rnn_b200.language_model import RecurrentLM, synthetic_text
from test_block import DTYPES, TINY, UNIT, logprobs_case, logprobs_exact, mlp_case, mlp_check, mlp_exact, near_in_norm, rand, within


# ---- log probabilities without logits: upstream gradients ------------------------------------------------------------------------

def logprobs_grads(x, w, t, up, **k):
    leaves = [v.detach().requires_grad_() for v in (x, w)]
    return torch.autograd.grad(fr.linear_logprobs(*leaves, t, **k), leaves, up)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [60, 300])
def test_upstream_gradients_of_ignored_rows(n, dtype):
    """What stands in the gradient of an ignored row's log probability changes no bit."""
    x, w, t, (g, h) = logprobs_case(n, 700, 64, dtype, seed=6)
    t[::3] = -100
    g = g * 1e-2
    g[::3] = 0
    want = logprobs_grads(x, w, t, [g, 1e-3 * h])
    assert all(v.any() for v in want)
    for there in (1.0, 1e8, 5e21, 1e30, math.inf, -math.inf, math.nan):
        other = g.clone()
        other[::3] = there
        assert all(torch.equal(a, b) for a, b in zip(logprobs_grads(x, w, t, [other, 1e-3 * h]), want)), there


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [60, 300])
def test_upstream_gradients_that_are_not_finite(n, dtype):
    """A row whose upstream gradients are infinite or NaN has no gradients; the other rows have those that they have beside zeros there."""
    x, w, t, up = logprobs_case(n, 700, 64, dtype, seed=7)
    up = [1e-5 * u for u in up]
    rows = torch.ones(n, dtype=torch.bool, device="cuda")
    rows[[4, 41]] = False
    for u in up:
        u[~rows] = 0
    want, _ = logprobs_grads(x, w, t, up)
    for k in range(2):
        for bad in (math.inf, math.nan):
            other = [u.clone() for u in up]
            other[k][~rows] = bad
            dx, _ = logprobs_grads(x, w, t, other)
            assert torch.equal(dx[rows], want[rows]) and not torch.isfinite(dx[~rows]).any()


# ---- products by clusters -----------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n,D,F,O", [(torch.bfloat16, 16, 4096, 12288, 64), (torch.float16, 30, 4096, 11000, 72), (torch.float32, 16, 4096, 12288, 64), (torch.float32, 1000, 2000, 2500, 300), (torch.float32, 300, 1024, 4096, 64)])
def test_clusters_with_several_tiles(dtype, n, D, F, O):
    """More tiles than clusters that run at once: a block's exchange buffer is used again, by its neighbours, after it has read it.  Right, and the
    same bits every time."""
    tensors, dy = mlp_case(n, D, F, O, dtype)
    want = mlp_check(tensors, dy)
    leaves = [v.requires_grad_() for v in tensors]
    for _ in range(20):
        y = fr.gated_mlp(*leaves)
        assert all(torch.equal(a, b) for a, b in zip([y, *torch.autograd.grad(y, leaves, dy)], want))


# ---- sums along k ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("k", [9000, 100000])
def test_long_sums_in_16_bits_lean_to_neither_side(k, dtype):
    """Accumulators truncate: a unit of the last place at most of the sum so far for each 16 values, in the mean half a unit of half the
    sum (and the products' own alignment, which of 8 by 11 bits loses hardly any).  That is 256 times 2^-25 in a part of 64 steps of 64 values, 2^-17 of the result, whatever k; without parts k / 16 times 2^-25, at 100000 1.9e-4.
    All terms here are positive, so that the loss is on one side and shows in the mean over the results.  These are not independent in their roundings:
    a row's results lie within k^-1/2 of one another, in bf16 less than a step (of 15 different x0 there is 3.4e-4 in the mean of the exact results'
    roundings alone).  So they are compared with the exact results rounded to the same type: of those a part s (steps a result) that lies within the shift
    from a border goes one step, which in the mean is the shift again, times at most 0.4 steps over the spread's k^-1/2 where a border cuts the middle of
    them (bf16, k = 100000: 1.0): 2^-16 is twice what the parts lose.  (The hidden vectors are exact: relu(1) times whole numbers up to 225.  There
    are results enough that k is not cut into slices.)"""
    n, D, O = 2100, 8, 2048
    g = torch.Generator(device="cuda").manual_seed(1)
    x, gate, up = (torch.zeros(m, D, device="cuda") for m in (n, k, k))
    x[:, 0], up[:, 0] = torch.randint(1, 16, (n,), generator=g, device="cuda"), torch.randint(1, 16, (k,), generator=g, device="cuda")
    x[:, 1], gate[:, 1] = 1.0, 1.0
    down = (torch.rand(O, k, generator=g, device="cuda") + 0.5) * 2.0 ** -10
    x, gate, up, down = (v.to(dtype) for v in (x, gate, up, down))
    y = fr.gated_mlp(x, gate, up, down, activation="relu").double()
    want = lm.naive_gated_mlp(*(v.double() for v in (x, gate, up, down)), "relu")
    assert abs(float(((y - want.to(dtype).double()) / want).mean())) <= 2.0 ** -16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [30, 300])
def test_gradients_of_confident_rows(n, dtype):
    """Tokens whose probability is near 1, from long sums: the gradient is in proportion to 1 - p, p = exp of the difference between a logit and the
    log of the sum, and loses 1 / (1 - p) times what the two disagree by.  Logits are sums of positive terms, about 40; in parts of 1024 values each is
    short by 2^-19 at most (64 times 2^-25, see above), so the two by 40 2^-19, and 1 - p = 1.2e-3 or more is off by 6.4 % at most."""
    D, V = 16384, 1000
    g = torch.Generator().manual_seed(4)
    x, w = torch.rand(n, D, generator=g) + 0.5, torch.rand(V, D, generator=g) + 0.5
    w *= 26.5 / D
    w[7] *= 40 / 26.5
    x, w = x.cuda().to(dtype), w.cuda().to(dtype)
    t = torch.full((n,), 7, device="cuda")
    leaves, exact = [v.requires_grad_() for v in (x, w)], [v.detach().double().requires_grad_() for v in (x, w)]
    got = torch.autograd.grad(fr.linear_logprobs(*leaves, t).logprob.sum(), leaves)
    r = lm.naive_linear_logprobs(*exact, t)
    assert 2e-4 < float(-r.logprob.detach().mean()) < 5e-3
    for a, b in zip(got, torch.autograd.grad(r.logprob.sum(), exact)):
        assert float((a.double() - b).norm()) <= 0.07 * float(b.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [5, 300, 3000])
def test_log_probabilities_near_zero(n, dtype):
    """The log probability of the likeliest token, -log(1 + rest), has the rounding of 1 + rest and an exponential's error of the rest, whatever the
    logits' size: logits are whole numbers here (width 1), exact in every type."""
    V = 700
    w = torch.zeros(V, 1, device="cuda")
    w[3], w[11] = 1.0, 0.875
    for size in (16.0, 64.0, 96.0, 200.0):
        x = torch.full((n, 1), size, device="cuda")
        r = fr.linear_logprobs(x.to(dtype), w.to(dtype), torch.full((n,), 3, device="cuda"))
        want = lm.naive_linear_logprobs(x.double(), w.double(), torch.full((n,), 3, device="cuda"))
        # rest = exp(-size / 8) + 698 exp(-size): 2^-24 of size for each of both logits' roundings after their factor, and of their difference's; 2^-21 of an exponential
        rest = math.exp(-size / 8)
        assert float((r.logprob.double() - want.logprob).abs().max()) <= 2.0 ** -22 + (size * 2.0 ** -22 + 2.0 ** -21) * rest


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,parts", [(1, 2.0 ** -19), (16, 2.0 ** -19), (128, 2.0 ** -19), (300, 2.0 ** -17)])
def test_logits_of_16_bit_operands(n, parts, dtype):
    """Long sums of positive terms.  An instruction loses two units of the last place at most (test_block), 2^-22 of the part's sum so far, which is half
    of the whole in the mean: 16 times 2^-23 in parts of 4 steps (up to 128 rows), 64 times in parts of 16.  Of two logits, z and 0, the log
    probability of the second is -log(1 + exp(z)), -z for z of 20."""
    D = 16384
    g = torch.Generator().manual_seed(5)
    x, w = (torch.rand(n, D, generator=g) + 0.5).cuda().to(dtype), torch.zeros(2, D)
    w[0] = (torch.rand(D, generator=g) + 0.5) * 20 / D
    w, t = w.cuda().to(dtype), torch.ones(n, dtype=torch.int64, device="cuda")
    want = lm.naive_linear_logprobs(x.double(), w.double(), t).logprob
    assert abs(float(((fr.linear_logprobs(x, w, t).logprob.double() - want) / want).mean())) <= parts


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [60, 300])
def test_gradients_at_the_least_temperature(n, dtype):
    """1 / T and fp16's factor for small gradients are each in range where their product is not.  Logits are 0: of x the weight's zeros see the only
    column that is not 0.  Errors in norm: UNIT for the rounding of the logits' gradient and of the result, and half of fp16's least number (2^-24) for each
    result that is not 0: the weight's gradients, sums of 3e-36 / T / 700 and the like, lie at that number."""
    x, w, t, up = logprobs_case(n, 700, 64, dtype, seed=11)
    x.zero_()
    x[:, 0] = 1
    w *= 32
    w[:, 0] = 0
    up = [3e-36 * u.clamp(-3, 3) for u in up]
    exact = [v.detach().double().requires_grad_() for v in (x, w)]
    T = float(torch.tensor(1e-30))
    want = torch.autograd.grad(lm.naive_linear_logprobs(*exact, t, T), exact, [u.double() for u in up])
    for a, b in zip(logprobs_grads(x, w, t, up, temperature=1e-30), want):
        assert float((a.double() - b).norm()) <= (2 * UNIT[dtype] + 2.0 ** -18) * float(b.norm()) + (TINY[dtype] / 2) * float((b != 0).sum()) ** 0.5


# ---- log probabilities without logits: memory -----------------------------------------------------------------------------------------

class Logprobs(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("token_bytes", ctypes.c_int32), *[(k, ctypes.c_int64) for k in ("n", "vocab", "width")], ("x", ctypes.c_void_p), ("weight", ctypes.c_void_p),
                ("x_stride", ctypes.c_int64), ("weight_stride", ctypes.c_int64), ("tokens", ctypes.c_void_p), ("ignore_index", ctypes.c_int64), ("temperature", ctypes.c_float)]


def test_workspace_of_the_forward_is_bounded():
    """What lies between the two kernels of a forward takes 256 MB at most (and 4 bytes a row), however many rows there are."""
    workspace = runtime.lib().frnn_linear_logprobs_forward_workspace
    workspace.restype = ctypes.c_size_t
    for n in (1, 300, 20000, 262144, 2 ** 24):
        for V in (1, 50257, 131072, 2 ** 20):
            size = workspace(ctypes.byref(Logprobs(1, 8, n, V, 64, 4096, 4096, 64, 64, 4096, -100, 1.0)))
            assert 0 < size <= 2 ** 28 + 2 ** 20 * 4 * 3 + 4 * n + 1024, (n, V, size)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_in_pieces(dtype):
    """More rows than a forward takes at once: those of both pieces have their own tokens, and the results that they have alone."""
    n, V, D = 15001, 100003, 24
    x, w, t, _ = logprobs_case(n, V, D, dtype)
    t[::7] = -100
    leaf = x.requires_grad_()
    r = fr.linear_logprobs(leaf, w, t)
    g = rand(n, seed=12)
    (dx,) = torch.autograd.grad(r.logprob, leaf, g)
    for lo in range(0, n, 1500):
        s = slice(lo, lo + 1500)
        want, tol = logprobs_exact(x.detach()[s], w, t[s], [g[s], torch.zeros_like(g[s])], 1.0, -100)
        for got, e, far in zip((r.logprob[s], r.entropy[s], dx[s]), want, tol):
            within(got, e, far)


@pytest.mark.gpu
def test_confident_rows_of_the_last_piece():
    """6500 rows against 2^20 tokens: the forward's last piece has 100 rows, and the backward takes them with all others.  Their gradients are in proportion to
    1 - p = 1e-3, and logits of 40, positive sums of 1024 terms, are short by up to 40 2^-17 in parts of 16 steps, 40 2^-19 in parts of 4: in both passes by the same, or
    gradients are off by a fifth.  (What is left: see test_gradients_of_confident_rows.)"""
    n, V, D = 6500, 2 ** 20, 1024
    g = torch.Generator(device="cuda").manual_seed(6)
    x, w = torch.rand(n, D, generator=g, device="cuda") + 0.5, torch.rand(V, D, generator=g, device="cuda") + 0.5
    w *= 19.5 / D
    w[7] *= 40 / 19.5
    x, w = x.half().requires_grad_(), w.half()
    t = torch.full((n,), 7, device="cuda")
    (dx,) = torch.autograd.grad(fr.linear_logprobs(x, w, t).logprob.sum(), x)
    for rows in (slice(0, 100), slice(n - 100, n)):
        z = (x.detach()[rows].double() @ w.double().T).requires_grad_()
        lp = lm.naive_token_logprobs(z, t[rows]).logprob
        assert 1e-4 < float(-lp.detach().mean()) < 1e-2
        G, = torch.autograd.grad(lp.sum(), z)
        want = G @ w.double()
        assert float((dx[rows].double() - want).norm()) <= 0.07 * float(want.norm())


# ---- the language model ---------------------------------------------------------------------------------------------------------------

def test_positions_go_on_with_the_states():
    """A text read in parts, each from the states of the one before, is the text read at once; a position that is given counts."""
    torch.manual_seed(1)
    model = RecurrentLM(97, width=48, layers=2, heads=3, head_width=16, plain=True, hidden=80, turned=12).double()
    text = synthetic_text(3, 20, 97)
    whole, _ = model(text)
    states, parts = None, []
    for part in text.split([1, 7, 1, 11], 1):
        logits, states = model(part, states)
        parts.append(logits)
    assert torch.allclose(whole, torch.cat(parts, 1), atol=1e-10)
    _, first = model(text[:, :9])
    for position in (None, 9):
        assert torch.allclose(model(text[:, 9:], first, position)[0], whole[:, 9:], atol=1e-10)
    assert not torch.allclose(model(text[:, 9:], first, 0)[0], whole[:, 9:], atol=1e-3)
    assert torch.equal(model(text, [s[:2] for s in model.states(3)])[0], whole)


def test_frequencies_move_with_the_model():
    for device in ("meta", "cpu"):
        for dtype in (torch.bfloat16, torch.float64):
            layer = RecurrentLM(97, width=48, layers=1, heads=3, head_width=16, turned=12).to(device, dtype).layers[0]
            assert layer.norm_weight.dtype == dtype and layer.frequencies.dtype == torch.float64 and layer.frequencies.device == layer.norm_weight.device
    layer = RecurrentLM(97, width=48, layers=1, heads=3, head_width=16, turned=12).to("meta").to_empty(device="cpu").layers[0]
    assert torch.equal(layer.frequencies, lm.rotary_frequencies(12, base=500.0))


@pytest.mark.gpu
def test_first_call_of_a_model_in_a_graph():
    """A model's first call is captured (the scan has been compiled before, by a model without positions)."""
    make = lambda turned: RecurrentLM(97, width=48, layers=2, heads=3, head_width=16, hidden=80, turned=turned, keep_logits=False).cuda().bfloat16()
    text = synthetic_text(4, 33, 97).clamp_min(0).cuda()
    with torch.no_grad():
        make(0).score(text)
        torch.cuda.synchronize()
        model = make(12)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = model.score(text)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, model.score(text)))


# ---- rotary positions -----------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("start", [0, 10 ** 6])
def test_rotations_in_fp32(start):
    """Errors in norm, in units of 2^-24, of which a rounding is 0.42 (half a unit of the last place at most, uniform, over mantissas): the result's, half of
    one for the product that is rounded, sine and cosine half a unit each: sqrt(0.42^2 (1 + 1 / 2) + 0.5^2) = 0.72.  The angle's rest adds nothing."""
    x, f = rand(1, 4096, 2, 128), lm.rotary_frequencies(128, device="cuda")
    for interleaved in (False, True):
        want = lm.naive_rotary(x.double(), start, f, interleaved)
        assert float((fr.rotary(x, start, f, interleaved).double() - want).norm()) <= 0.75 * 2.0 ** -24 * float(want.norm())


# ---- fp32 ------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("n,D,F,O,product", [(16, 1024, 2048, 1024, 3e-7), (300, 520, 1300, 520, 1e-6), (1000, 512, 2048, 512, 1e-6), (4096, 256, 3840, 256, 3e-7), (2048, 1024, 4096, 1024, 3e-7)])
def test_products_of_fp32_in_norm(n, D, F, O, product):
    """Errors in norm that show each of the six products of planes: without (lo, hi) or (hi, lo) a product is off by 2.4e-6.  An instruction loses two units of
    the last place at most, 0.72 2^-22 of the part's sum so far, which of terms of either sign grows with the square root: of m instructions 2 / 3 m times
    that.  Steps of six products have 4 of the largest planes, behind the small ones: 3e-7 (few rows; pairs of blocks; blocks alone, with slices of k);
    clusters of more rows have parts of 16: 1e-6.  A result has two (y, down's gradient) or three products on its way, and 2^-21 for the activation and roundings."""
    tensors, dy = mlp_case(n, D, F, O, torch.float32, seed=13)
    leaves, exact = [v.requires_grad_() for v in tensors], [v.detach().double().requires_grad_() for v in tensors]
    y, want = fr.gated_mlp(*leaves), lm.naive_gated_mlp(*exact)
    for a, b, products in zip([y, *torch.autograd.grad(y, leaves, dy)], [want, *torch.autograd.grad(want, exact, dy.double())], (2, 3, 3, 3, 2)):
        assert float((a.double() - b).norm()) <= (products * product + 2.0 ** -21) * float(b.norm())


@pytest.mark.gpu
@pytest.mark.parametrize("n,V,D", [(16, 5003, 1024), (300, 3001, 485), (2000, 9001, 256), (130, 777, 2000)])
def test_log_probabilities_of_fp32_in_norm(n, V, D):
    """As above.  Logits of some units (in norm sqrt(2) times a log probability's error at most): one product of either kind; gradients a second one, and p with a
    logit's error, 2 times its size, in forward and backward."""
    x, w, t, up = logprobs_case(n, V, D, torch.float32, seed=13)
    leaves, exact = [v.requires_grad_() for v in (x, w)], [v.detach().double().requires_grad_() for v in (x, w)]
    r, want = fr.linear_logprobs(*leaves, t), lm.naive_linear_logprobs(*exact, t)
    for a, b in zip(r, want):
        assert float((a.double() - b).norm()) <= (1.5e-6 + 2.0 ** -21) * float(b.norm())
    for a, b in zip(torch.autograd.grad(r, leaves, up), torch.autograd.grad(want, exact, [u.double() for u in up])):
        assert float((a.double() - b).norm()) <= (1e-6 + 4e-6 + 2.0 ** -21) * float(b.norm())


# ---- log probabilities without logits: pieces, planes -----------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n,V,D", [(torch.float32, 1000, 150000, 64), (torch.float32, 2000, 150000, 200), (torch.float16, 600, 600000, 40), (torch.bfloat16, 700, 500000, 40)])
def test_pieces_of_a_long_vocabulary(dtype, n, V, D):
    """Few rows against a vocabulary in pieces: x's gradient is added up over pieces and, in each, over slices of it."""
    x, w, t, up = logprobs_case(n, V, D, dtype)
    leaves = [v.requires_grad_() for v in (x, w)]
    got = torch.autograd.grad(fr.linear_logprobs(*leaves, t), leaves, up)
    want, tol = logprobs_exact(x.detach(), w.detach(), t, up, 1.0, -100)
    for g, e, far in zip(got, want[2:], tol[2:]):
        within(g, e, far)
        near_in_norm(g, e, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,every", [(128, 16), (129, 16), (200, 25), (2000, 100)])
def test_few_rows_that_count(n, every, dtype):
    """Most rows ignored: up to 128 rows in two planes of the logits' gradient, above in one, whose rounding is that of the results again."""
    x, w, t, (g, h) = logprobs_case(n, 3000, 383, dtype, seed=14)
    ignored = torch.arange(n, device="cuda") % every != 3
    t[ignored] = -100
    h[ignored] = 0
    for got, e, far in zip(logprobs_grads(x, w, t, [g, h]), *(v[2:] for v in logprobs_exact(x, w, t, [g, h], 1.0, -100))):
        within(got, e, far)
        near_in_norm(got, e, 1 if n <= 128 else 2)


# ---- large ones -----------------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,D,F,O", [(20, 9000, 300, 4400), (600, 4500, 1300, 4200), (2100, 4300, 1500, 8300)])
def test_gated_mlp_of_wide_models(n, D, F, O, dtype):
    """More than 64 steps of k in the products whose results the activation takes, alone, in clusters and by pairs."""
    mlp_check(*mlp_case(n, D, F, O, dtype, seed=15))


@pytest.mark.gpu
def test_gated_mlp_offsets_past_31_bits():
    """2.2 10^9 hidden values; all rows but the last ones are zero, and add nothing to the gradients of the weights."""
    n, last, (D, F, O) = 131100, 60, (16, 16500, 24)
    (x, *weights), dy = mlp_case(last, D, F, O, torch.bfloat16, seed=16)
    wide, far = torch.zeros(n, D, dtype=x.dtype, device="cuda"), torch.zeros(n, O, dtype=x.dtype, device="cuda")
    wide[-last:], far[-last:] = x, dy
    leaves = [v.requires_grad_() for v in (wide, *weights)]
    y = fr.gated_mlp(*leaves)
    dx, *dw = torch.autograd.grad(y, leaves, far)
    want, tol = mlp_exact(x, *(v.detach() for v in weights), dy, "silu")
    assert not y[:-last].any() and not dx[:-last].any()
    for got, e, t in zip((y[-last:], dx[-last:], *dw), want, tol):
        within(got, e, t)


@pytest.mark.gpu
def test_linear_logprobs_offsets_past_31_bits():
    """A weight of 2.5 10^9 elements, of which only the last rows are not zero: the other tokens' logits are 0, and their probabilities equal."""
    n, V, D, last = 20, 300000, 8192, 3000
    x, w, _, (g, h) = logprobs_case(n, last, D, torch.float16, seed=17)
    t = V - 1 - 7 * torch.arange(n, device="cuda")
    big = torch.zeros(V, D, dtype=w.dtype, device="cuda")
    big[-last:] = w
    leaves = [v.requires_grad_() for v in (x, big)]
    r = fr.linear_logprobs(*leaves, t)
    dx, dw = torch.autograd.grad(r, leaves, [g, h])
    z = torch.cat([torch.zeros(n, 1, device="cuda", dtype=torch.float64), x.detach().double() @ w.double().T], 1).requires_grad_()      # (column 0: each of the others)
    many = torch.ones(last + 1, device="cuda", dtype=torch.float64)
    many[0] = V - last
    lse = torch.log((many * z.exp()).sum(-1, True))
    p = (z - lse).exp()
    lp, H = (z - lse).gather(1, (t - (V - last) + 1)[:, None])[:, 0], -(many * p * (z - lse)).sum(-1)
    G, = torch.autograd.grad([lp, H], z, [g.double(), h.double()])
    G = G / many
    ez = 2.0 ** -19 * float((x.detach().double().abs() @ w.double().abs().T).max()) + 2.0 ** -20          # (a logit's error in parts of 4 steps; exponentials)
    assert float((r.logprob.double() - lp.detach()).abs().max()) <= 2 * ez and float((r.entropy.double() - H.detach()).abs().max()) <= 2 * ez * (1 + math.log(V))
    u = UNIT[w.dtype]
    for got, e, size in ((dx, G[:, 1:] @ w.double(), G[:, 1:].abs() @ w.double().abs()), (dw[-last:], G[:, 1:].T @ x.detach().double(), G[:, 1:].abs().T @ x.detach().double().abs()),
                         (dw[:1000], (G[:, :1].T @ x.detach().double()).expand(1000, D), (G[:, :1].abs().T @ x.detach().double().abs()).expand(1000, D))):
        within(got, e, u * size)
