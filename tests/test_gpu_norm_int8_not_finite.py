"""Rows with infinities and NaNs through the int8 norm: their scale is NaN whatever the
rotation, the weight or the other values make of them."""

import math

import pytest
import torch

from mx_util import DTYPES, randn
from xpu_kernels import int8, norm

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


def rows(k):
    """The rows to spoil, and the weight's places that are 0"""
    one, four, mixed, nans, far = (randn(k, seed=i) for i in range(5))
    one[k // 2] = INF
    q = 4 * (k // 8)                                   # a quartet that the rotation sums and subtracts
    four[q:q + 4] = INF
    mixed[::2], mixed[1::2] = INF, -INF
    nans[k - 1] = NAN
    far[0] = -INF                                      # where the weight is 0
    return torch.stack([torch.full((k,), INF), torch.full((k,), -INF), one, four, mixed, nans, far])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rotate,k", [(True, k) for k in (256, 768, 1280, 4096, 16384, 16640, 33024)] +
                         [(False, k) for k in (5, 64, 100, 1000, 1280, 5120, 20000, 33024, 40001)])
@pytest.mark.parametrize("residual", [False, True])
def test_scales_of_rows_that_are_not_finite(dev, dtype, rotate, k, residual):
    bad = rows(k).to(dtype)
    good = randn(3, k, seed=9).to(dtype)
    x = torch.stack([v for pair in zip(bad, good.repeat(3, 1)) for v in pair])     # bad and good in turn
    w = 1 + 0.2 * randn(k, seed=3)
    w[0] = 0.0
    r = randn(len(x), k, seed=4).to(dtype).to(dev) if residual else None
    for weight in (None, w.to(dev)):
        q, s, *_ = norm.rms_norm_int8(x.to(dev), weight, residual=r, rotate=rotate)
        assert s[::2].isnan().all(), s[::2]
        clean = norm.rms_norm_int8(x[1::2].to(dev), weight, residual=None if r is None else r[1::2], rotate=rotate)
        assert torch.equal(q[1::2], clean[0]) and torch.equal(s[1::2], clean[1]) and s[1::2].isfinite().all()


@pytest.mark.parametrize("rotate,k", [(True, 256), (True, 1280), (True, 16640), (False, 40), (False, 2048), (False, 40000)])
def test_a_weight_that_is_not_a_number(dev, rotate, k):
    x, w = randn(4, k, seed=1).to(dev), 1 + 0.2 * randn(k, seed=3)
    w[k // 3] = NAN
    assert norm.rms_norm_int8(x, w.to(dev), rotate=rotate)[1].isnan().all()


@pytest.mark.parametrize("rotate,k", [(True, 256), (True, 1280), (True, 16640), (False, 40), (False, 2048), (False, 40000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_finite_rows_whose_squares_overflow(dev, dtype, rotate, k):
    """Zeros, as rms_norm's."""
    x = (randn(4, k, seed=1) * 1e25).to(dtype).to(dev)
    assert not norm.rms_norm(x).any()
    assert not norm.rms_norm_int8(x, rotate=rotate)[1].any()


def test_an_overflow_reaches_the_linear(dev):
    """An fp16 residual stream that overflows everywhere is not hidden by the codes."""
    x = torch.full((2, 512), 60000.0, dtype=torch.float16, device=dev)
    w8, ws = int8.prepare_weight(randn(64, 512, seed=1).bfloat16().to(dev))
    q, s, h = norm.rms_norm_int8(x, residual=x)
    assert h.isinf().all() and s.isnan().all()
    assert int8.linear_quantized(q, s, w8, ws).isnan().all()
