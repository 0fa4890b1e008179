"""Calls of gated_mlp, linear_logprobs and rotary (flex_rnn_b200.lm) at their edges; tolerances are those of test_block."""
import math

import pytest
import torch

import flex_rnn_b200 as fr
from flex_rnn_b200 import lm
from test_block import DTYPES, logprobs_case, mlp_case, mlp_check


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
