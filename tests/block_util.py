"""Shared by the tests of RMS norm, routing and rotary positions: error bounds."""

import torch

from mx_util import HALF_TINY, HALF_ULP

#: half an fp32 unit in the last place, relative
U = 2.0 ** -24


def within(got, want, error):
    """|got - want| <= error before the one rounding to got's type."""
    g = got.detach().cpu().double()
    assert g.shape == want.shape, (g.shape, want.shape)
    bound = error + HALF_ULP[got.dtype] * (want.abs() + error) + HALF_TINY[got.dtype]
    bad = ~((g - want).abs() <= bound) & ~(g.isnan() & want.isnan()) & ~(g == want)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} outside the bound, first at "
                           f"{torch.nonzero(bad)[0].tolist()}: {g[bad][0]} for {want[bad][0]}, "
                           f"bound {bound.expand_as(bad)[bad][0]}")


def chain(k):
    """The most fp32 additions that one term of a row's sum goes through: 32 values of a lane
    one after another (rows over 32768: 8 of every 8192), 6 across a wave, 16 waves (64
    partial sums in the rotated form)."""
    return max(32, 8 * -(-k // 8192)) + 6 + 64


def norm_error(k):
    """Relative error of 1 / rms in fp32: the sum's, halved by the root, and the roundings of
    the mean, eps' addition, the root and the division."""
    return (chain(k) / 2 + 4) * U
