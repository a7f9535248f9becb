"""Routing where logits or biases are NaN or infinite: what is chosen, and the gradient."""

import math

import pytest
import torch

import oracle.block as O
from mx_util import DTYPES, randn
from xpu_kernels import moe

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e,groups,tokens", [(16, 2, 3), (64, 4, 3), (256, 8, 3), (1024, 8, 3), (64, 4, 65600)])
def test_a_group_of_nan_keys_comes_before_one_with_nothing(dev, dtype, scores, e, groups, tokens):
    """A NaN key is the lowest, but may be chosen: not before any other, and before none at all."""
    n = e // groups
    logits = randn(1, e, seed=1).to(dtype)
    logits[0, :n] = -math.inf                          # the first group: nothing to choose from
    bias = torch.full((e,), math.nan)
    how = dict(scores=scores, groups=groups, top_groups=1)
    ids, w = moe.route(logits.to(dev).expand(tokens, -1), 2, bias=bias.to(dev), **how)
    assert (ids.cpu() == torch.tensor([n, n + 1])).all()       # the second group, by index
    assert w.isfinite().all()
    oid, _ = O.route(logits, 2, bias=bias, **how)
    assert torch.equal(ids[:1].cpu(), oid)
    # one NaN and one finite key, in the last group, are above two NaNs
    bias[-1] = -1.0
    ids, _ = moe.route(logits.to(dev).expand(tokens, -1), 2, bias=bias.to(dev), **how)
    assert (ids.cpu() == torch.tensor([e - 1, e - n])).all()
    oid, _ = O.route(logits, 2, bias=bias, **how)
    assert torch.equal(ids[:1].cpu(), oid)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_a_token_of_nans_beside_a_masked_group(dev, dtype, scores):
    """The same for a row whose logits are NaN: valid experts, weights of NaN."""
    logits = torch.full((4, 32), math.nan, dtype=dtype)
    logits[:, :8] = -math.inf
    logits[1] = randn(32, seed=3).to(dtype)
    how = dict(scores=scores, groups=4, top_groups=1)
    ids, w = moe.route(logits.to(dev), 3, **how)
    oid, _ = O.route(logits, 3, **how)
    assert torch.equal(ids.cpu(), oid) and (ids >= 0).all()
    assert w[[0, 2, 3]].isnan().all() and w[1].isfinite().all()
