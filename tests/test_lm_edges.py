"""Calls of the operators around the scans (flex_rnn_b200.lm) at their edges; tolerances are those of test_lm."""
import math

import pytest
import torch

import flex_rnn_b200 as fr
from test_lm import DTYPES


# ---- log probabilities: NaN --------------------------------------------------------------------------------------------------

def short_row(dtype):
    """The longest row that one warp takes where there are rows enough."""
    return 8192 // torch.finfo(dtype).bits * 8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V", [(3, 9001), (3, 70000), (400, 40000), (1300, 0)])
def test_nan_among_masked_logits(n, V, dtype):
    """A NaN makes its row NaN whatever follows it: rows whose other logits are all -inf, or nearly all, with the NaN in the
    first loads of a thread that has more of them.  Rows of nothing but -inf stay what they are."""
    V = V or short_row(dtype) - 3
    x = torch.full((n, V), -math.inf, dtype=dtype, device="cuda")
    t = torch.full((n,), 5, device="cuda")
    at = [3, 0]
    for row in range(n):
        if row % 3 != 2:
            x[row, at[row % 3]] = math.nan
    x[1, 7] = 1.5
    leaf = x.requires_grad_()
    r = fr.token_logprobs(leaf, t, top=4)
    g = torch.autograd.grad((r.logprob, r.entropy), leaf, (torch.ones(n, device="cuda"), torch.ones(n, device="cuda")))[0]
    bad = torch.arange(n, device="cuda") % 3 != 2
    for v in (r.logprob, r.entropy):
        assert torch.equal(v.isnan(), bad)
    assert torch.equal(r.top_logprob.isnan().all(1), bad) and torch.equal(g.isnan().all(1), bad)
    assert (r.logprob[~bad] == -math.inf).all() and not r.entropy[~bad].any() and not g[~bad].any()
    assert r.top_token[0].tolist() == [3, 0, 1, 2] and r.top_token[1].tolist() == [0, 7, 1, 2] and r.top_token[2].tolist() == [0, 1, 2, 3]
