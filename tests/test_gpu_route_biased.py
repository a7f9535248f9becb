"""Softmax keys with a bias: a small score with a large bias next to a large score.  The
error of the scores' sum moves such keys apart, where those of near scores move together."""

import math

import pytest
import torch

import oracle.block as O
from mx_util import DTYPES, randn
from xpu_kernels import moe

pytestmark = pytest.mark.gpu

#: experts, groups, groups kept, tokens: 8, 16, 32 and 64 lanes a token, of 4 to 32 experts
#: each, with the lanes of few tokens and of many
LANES = [(64, 1, 1, 1), (100, 1, 1, 1), (256, 1, 1, 1), (60, 4, 4, 1), (256, 8, 4, 1),
         (256, 8, 4, 65536), (384, 1, 1, 1), (384, 1, 1, 8192), (1000, 1, 1, 1), (1000, 1, 1, 8192)]


def pair(e, dtype, seed, small, large):
    """(logits [1, e], bias [e]): the expert `small` has a tiny score and a bias that brings its
    key to within a unit or two of the score of `large`."""
    logits = randn(1, e, seed=seed).to(dtype)
    logits[0, small] = -12.0
    logits[0, large] = math.log(e) + 0.25 * (seed % 5)
    s = torch.softmax(logits.double(), -1)[0]
    bias = torch.zeros(e)
    bias[small] = (s[large] - s[small]).float()
    for _ in range(seed % 3):                        # the fp32 number nearest to it, or one beside it
        bias[small] = torch.nextafter(bias[small], torch.tensor(float(seed % 2)))
    return logits, bias


def check(dev, logits, bias, top, tokens, **how):
    want, _ = O.route(logits, top, bias=bias, **how)
    ids, _ = moe.route(logits.to(dev).expand(tokens, -1), top, bias=bias.to(dev), **how)
    return bool((ids.cpu() == want).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("e,groups,top_groups,tokens", LANES)
@pytest.mark.parametrize("renormalize", [True, False])
def test_a_small_score_beside_a_large_one(dev, dtype, e, groups, top_groups, tokens, renormalize):
    """Both within the chosen ones, and on either side of the last."""
    wrong = []
    for seed in range(24 if tokens == 1 else 6):
        g = torch.Generator().manual_seed(seed)
        n = e // groups
        a, b = torch.randperm(n, generator=g)[:2].sort().values.tolist()
        small, large = (a, b) if seed % 4 else (b, a)
        logits, bias = pair(e, dtype, seed, small, large)
        for top in (1, 2, 8):
            if not check(dev, logits, bias, top, tokens, groups=groups, top_groups=top_groups,
                         renormalize=renormalize):
                wrong.append((seed, top))
    assert not wrong, wrong


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [0.99999696, 0.99999642, 0.9999971])
def test_many_small_scores(dev, dtype, bias):
    """Exponentials whose fp32 sum rounds up, one after another, in one lane; every logit is
    whole in 16 bits."""
    logits = torch.full((1, 256), -80.0)
    logits[0, :32] = -16.375
    logits[0, 1] = 0.0
    b = torch.zeros(256)
    b[0] = bias
    for top in (1, 2, 8):
        assert check(dev, logits.to(dtype), b, top, 1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_only_by_rounding(dev, dtype):
    """A key that meets another one in 64 bits with the fp32 sum, and not with the exact one, is
    no tie: many biases beside one score."""
    for e in (64, 256):
        wrong = 0
        for seed in range(40):
            logits, bias = pair(e, dtype, seed, 3, 40)
            s = torch.softmax(logits.double(), -1)[0]
            bias[3] = (s[40] - s[3]).float()
            wrong += not check(dev, logits, bias, 1, 1)
        assert not wrong, (e, wrong)
