"""Shared by the MXFP4 and mixture-of-experts tests: inputs and error bounds."""

import pytest
import torch


@pytest.fixture
def big_memory():
    """For a test of several GiB: its memory goes back to the device afterwards, so that
    no later test's allocation keeps a segment of it."""
    yield
    torch.cuda.empty_cache()


#: half a unit in the last place, relative (2^-p for p significant bits: 8, 11, 24)
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
#: the least subnormal's half (rounding below the normal range), absolute
HALF_TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def assert_close(got, want, magnitude, terms):
    """|got - want| is within what ``terms`` fp32 additions (each at most an ulp, 2^-23,
    of the running sum, itself at most ``magnitude`` = the sum of the terms'
    magnitudes) and one rounding to got's type can make."""
    g = got.detach().cpu().double()
    assert g.shape == want.shape
    u = HALF_ULP[got.dtype]
    acc = terms * 2.0 ** -23 * magnitude
    bound = acc + u * (want.abs() + acc) + HALF_TINY[got.dtype]
    bad = ~((g - want).abs() <= bound) & ~(g.isnan() & want.isnan()) & ~(g == want)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} outside the bound, first at "
                           f"{torch.nonzero(bad)[0].tolist()}: {g[bad][0]} for {want[bad][0]}")


def router(t, top, experts, seed=0, dropped=0.0, dtype=torch.int32):
    """Distinct experts a token (more slots than experts: repeats), some slots -1."""
    g = torch.Generator().manual_seed(seed)
    score = torch.randn(t, experts, generator=g) + torch.randn(experts, generator=g)
    ids = score.topk(min(top, experts), dim=-1).indices
    if top > experts:
        ids = torch.cat([ids] * -(-top // experts), 1)[:, :top]
    ids = torch.where(torch.rand(t, top, generator=g) < dropped, -1, ids)
    return ids.to(dtype)
