"""The gradient of routing for tokens whose logits make their weights NaN."""

import math

import pytest
import torch

import oracle.block as O
from mx_util import DTYPES, randn
from xpu_kernels import moe

pytestmark = pytest.mark.gpu

HOWS = [dict(), dict(renormalize=False), dict(scores="sigmoid"), dict(scores="sigmoid", renormalize=False)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", range(len(HOWS)))
@pytest.mark.parametrize("t,e,top", [(7, 8, 2), (9, 40, 4), (70, 64, 8), (6, 160, 6), (8, 256, 16), (6, 512, 8), (6, 1000, 8),
                                     (9, 40, 20), (6, 300, 32), (5, 1024, 64)])
def test_a_token_of_nan_weights_has_nan_gradients(dev, dtype, how, t, e, top):
    """Also where what made them NaN is not among the chosen; the other tokens' stay as they were."""
    how, soft = HOWS[how], HOWS[how].get("scores", "softmax") == "softmax"
    logits, dw = randn(t, e, seed=1).to(dtype), randn(t, top, seed=2).to(dev)

    def grad(v):
        x = v.to(dev).requires_grad_()
        ids, w = moe.route(x, top, **how)
        return ids, w, torch.autograd.grad(w, x, dw)[0]

    _, _, clean = grad(logits)
    low = logits[0].argmin()
    logits[0, low] = math.nan                          # NaNs come last: not among the chosen
    logits[1, e // 2] = math.inf
    logits[2] = math.nan
    logits[3, 0], logits[3, e - 1] = -math.inf, math.nan
    ids, w, d = grad(logits)
    assert not (ids[0] == low).any()
    for row, spoilt in ((0, True), (1, soft), (2, True), (3, True)):
        assert bool(w[row].isnan().all()) == spoilt
        assert bool(d[row].isnan().all()) == spoilt and bool(d[row].isnan().any()) == spoilt, row
    assert torch.equal(d[4:], clean[4:])
    want = O.route_grad(logits, ids.cpu(), dw.cpu(), **how)
    assert torch.equal(d.isnan().cpu(), want.isnan())


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_an_infinite_logit_outside_of_the_chosen_groups(dev, scores):
    """Behind a bias that keeps its group out."""
    logits = randn(5, 32, seed=1)
    logits[2, 30] = math.inf
    bias = torch.zeros(32)
    bias[24:] = -math.inf
    x = logits.to(dev).requires_grad_()
    ids, w = moe.route(x, 4, scores=scores, bias=bias.to(dev), groups=4, top_groups=2)
    d, = torch.autograd.grad(w.sum() + (w * w).sum(), x)
    soft = scores == "softmax"
    assert bool(w[2].isnan().all()) == soft and bool(d[2].isnan().all()) == soft
    assert d[[0, 1, 3, 4]].isfinite().all() and bool(d[2].isfinite().all()) != soft
