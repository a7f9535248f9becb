"""The choice of experts on the device against the 64-bit oracle: ids equal, weights and
gradients within their roundings."""

import math

import pytest
import torch

import oracle.block as O
from block_util import U, within
from mx_util import DTYPES, randn
from xpu_kernels import moe

pytestmark = pytest.mark.gpu

HOWS = [dict(), dict(renormalize=False), dict(scores="sigmoid"), dict(scores="sigmoid", scale=2.5),
        dict(scores="sigmoid", renormalize=False, scale=0.5), dict(renormalize=False, scale=-3.0)]


def logits_of(t, e, dtype, seed=1):
    return (randn(t, e, seed=seed) * 1.5 + randn(e, seed=seed + 1) * 0.5).to(dtype)


def weight_error(how):
    """Scores are 64 bits until their one rounding, but that a softmax's sum over all experts
    (which drops out of renormalised weights) may be fp32: of exponentials off by 2 units and
    by their argument's two roundings, |x| units each (their mean over the sum, e^-|x| |x| /
    e^-|x|, is under 8), 32 in a lane and 6 across lanes: 2 + 2 * 8 + 38 units."""
    return 56 * U if how.get("scores", "softmax") == "softmax" and not how.get("renormalize", True) else 1e-12


def check(dev, logits, top, dweights=None, **how):
    bias = how.get("bias")
    call = dict(how, bias=None if bias is None else bias.to(dev))
    lg = logits.to(dev).requires_grad_(dweights is not None)
    ids, w = moe.route(lg, top, **call)
    oid, ow = O.route(logits, top, **how)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(ids.cpu(), oid)
    within(w, ow, weight_error(how) * ow.abs())
    if dweights is None:
        return ids, w
    d, = torch.autograd.grad(w, lg, dweights.to(dev))
    kind = {k: v for k, v in how.items() if k in ("scores", "renormalize", "scale")}
    want = O.route_grad(logits, oid, dweights, **kind)
    # scale s (g - sum g s), a score to a sum of 64 or E exponentials, each in fp32 to a few
    # units, and the sum along g: bounded by the terms' magnitudes
    live = oid >= 0
    g = torch.where(live, dweights.double(), 0.0).abs()
    s = torch.softmax(logits.double(), -1).nan_to_num(0.0)
    part = torch.zeros_like(s).scatter_(1, oid.clamp(min=0).long(), torch.where(live, ow.abs(), 0.0))
    along = (g * torch.where(live, ow.abs(), 0.0)).sum(-1, keepdim=True)
    own = torch.zeros_like(s).scatter_add_(1, oid.clamp(min=0).long(), g * live)
    scale = abs(how.get("scale", 1.0))
    within(d, want, 40 * U * (part * (own + along / max(scale, 1e-30)) + scale * s * along / max(scale, 1e-30)))
    return ids, w


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", range(len(HOWS)))
@pytest.mark.parametrize("t,e,top", [(1, 1, 1), (1, 8, 2), (3, 5, 5), (67, 64, 8), (33, 65, 6),
                                     (9, 128, 1), (40, 160, 6), (35, 256, 8), (5, 300, 32),
                                     (4, 512, 64), (3, 1000, 8), (2, 1024, 64)])
def test_choice_and_gradient(dev, dtype, how, t, e, top):
    logits = logits_of(t, e, dtype)
    dw = randn(t, top, seed=7)
    check(dev, logits, top, dw, **HOWS[how])
    check(dev, logits, top, dw, **HOWS[how], bias=randn(e, seed=5) * 0.05)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", range(len(HOWS)))
@pytest.mark.parametrize("t,e,groups,top_groups,top", [
    (40, 64, 8, 4, 8), (9, 256, 8, 4, 8), (7, 160, 8, 3, 6), (5, 60, 4, 1, 4), (3, 30, 15, 2, 4),
    (4, 64, 64, 5, 5), (6, 1000, 10, 3, 9), (3, 1024, 64, 64, 16), (5, 24, 3, 3, 24), (2, 64, 2, 1, 32)])
def test_groups(dev, dtype, how, t, e, groups, top_groups, top):
    logits, dw = logits_of(t, e, dtype), randn(t, top, seed=7)
    for bias in (None, randn(e, seed=5) * 0.05):
        check(dev, logits, top, dw, **HOWS[how], groups=groups, top_groups=top_groups, bias=bias)


@pytest.mark.parametrize("how", range(len(HOWS)))
def test_many_tokens(dev, how):
    """Near and equal keys among many tokens."""
    for dtype, bias in ((torch.bfloat16, torch.zeros(64)), (torch.bfloat16, None),
                        (torch.float32, randn(64, seed=5) * 0.05)):
        check(dev, logits_of(3001, 64, dtype), 8, randn(3001, 8, seed=7), **HOWS[how], bias=bias)
        check(dev, logits_of(1501, 64, dtype), 6, **HOWS[how], bias=bias, groups=8, top_groups=3)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_ties_and_neighbours(dev, scores):
    """Equal keys go to the lower index; keys a few units of fp32 apart are told apart."""
    e = 96
    same = torch.zeros(3, e)
    same[1, 40:] = 1.0
    check(dev, same, 8, scores=scores)
    check(dev, same, 8, scores=scores, bias=torch.zeros(e))
    check(dev, same, 8, scores=scores, bias=torch.zeros(e), groups=8, top_groups=2)
    # scores one unit apart, in an order that the bias alone reverses
    near = torch.ones(4, e)
    near[:, ::3] = 1.0 + 2.0 ** -23
    near[2] = torch.nextafter(torch.full((e,), 0.5), torch.tensor(1.0)) + torch.arange(e) * 2.0 ** -24
    check(dev, near, 12, scores=scores)
    for step in (2.0 ** -26, 2.0 ** -30, 2.0 ** -40):
        bias = (torch.arange(e).flip(0) % 7).float() * step
        check(dev, near, 12, scores=scores, bias=bias)
        check(dev, near, 12, scores=scores, bias=bias, groups=4, top_groups=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", range(len(HOWS)))
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (8, 3)])
def test_masks(dev, dtype, how, bias, groups, top_groups):
    """Masked experts are never chosen, also when that leaves slots or the row empty."""
    t, e, top = 12, 64, 8
    logits = logits_of(t, e, dtype)
    logits[0] = -math.inf
    logits[1, 5:] = -math.inf
    logits[2, :-1] = -math.inf
    logits[3, ::2] = -math.inf
    logits[4, 8:] = -math.inf
    logits[5] = torch.where(torch.arange(e) % 8 == 3, logits[5], torch.tensor(-math.inf, dtype=dtype))
    logits[6] = torch.finfo(dtype).min                 # as masks write it: an ordinary value
    logits[7, 9:] = torch.finfo(dtype).min
    dw = randn(t, top, seed=7)
    b = None
    if bias:
        b = randn(e, seed=5) * 0.05
        b[17] = -math.inf                              # an expert that is switched off
    how = dict(HOWS[how], groups=groups, top_groups=top_groups, bias=b)
    dw[torch.arange(t)[:, None].expand(t, top) == 0] = math.nan     # of slots without an expert
    ids, w = check(dev, logits, top, dw, **how)
    assert (ids[0] == -1).all() and (w[0] == 0).all()
    # and sorting gives those slots to no expert
    assert int(moe.sort(ids, e).offsets[-1]) == int((ids >= 0).sum())


@pytest.mark.parametrize("how", range(len(HOWS)))
def test_not_finite(dev, how):
    """A row with a NaN has NaN weights of valid experts, the others as they were."""
    t, e, top = 6, 40, 4
    logits = logits_of(t, e, torch.float32)
    clean = moe.route(logits.to(dev), top, **HOWS[how])
    logits[1, 3] = math.nan
    logits[2] = math.nan
    logits[3, 7] = math.inf
    ids, w = check(dev, logits, top, **HOWS[how])
    soft = HOWS[how].get("scores", "softmax") == "softmax"
    assert w[1].isnan().all() and w[2].isnan().all() and bool(w[3].isnan().all()) == soft
    assert ((ids >= 0) & (ids < e)).all()
    rest = [0, 4, 5]
    assert torch.equal(ids[rest], clean[0][rest]) and torch.equal(w[rest], clean[1][rest])


@pytest.mark.parametrize("how", range(len(HOWS)))
def test_extremes(dev, how):
    """Scores far below what fp32 holds still make weights; saturated ones keep their order."""
    x = torch.stack([torch.linspace(-900, -600, 32), torch.linspace(30, 300, 32),
                     torch.linspace(-3e38, 3e38, 32), torch.linspace(-100, 100, 32)])
    ids, w = moe.route(x.to(dev), 4, **HOWS[how])
    oid, ow = O.route(x, 4, **HOWS[how])
    assert torch.equal(ids.cpu(), oid)
    within(w, ow, weight_error(HOWS[how]) * ow.abs())
    xg = x.to(dev).requires_grad_()
    d, = torch.autograd.grad(moe.route(xg, 4, **HOWS[how])[1], xg, torch.ones(4, 4, device=dev))
    # (fp32's linspace overflows over the third row's range: infinities and NaNs in it)
    assert torch.isfinite(x).all(-1).tolist() == [True, True, False, True]
    assert torch.isfinite(d[[0, 1, 3]]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dev, dtype):
    wide = logits_of(50, 90, dtype).to(dev)
    for lg in (wide[:, 5:69], wide[::3, 1:60], wide.t(), wide[:1].expand(7, 90), wide[:1, :3]):
        top = min(3, lg.shape[1])
        want = moe.route(lg.contiguous(), top)
        got = moe.route(lg, top)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        a, b = lg.detach().clone().requires_grad_(), lg.detach().requires_grad_()
        dw = randn(lg.shape[0], 2 * top, seed=3).to(dev)[:, ::2]
        ga, = torch.autograd.grad(moe.route(a, top)[1], a, dw)
        gb, = torch.autograd.grad(moe.route(b, top)[1], b, dw.contiguous())
        assert torch.equal(ga, gb)
    lg = wide[:0].clone().requires_grad_()
    ids, w = moe.route(lg, 4)
    assert ids.shape == w.shape == (0, 4)
    g, = torch.autograd.grad(w, lg, w)
    assert g.shape == (0, 90)
    bias = randn(90, seed=4)
    for b in (bias.half(), bias.bfloat16(), torch.stack([bias, bias], 1)[:, 0]):
        got, want = moe.route(wide, 4, bias=b.to(dev)), moe.route(wide, 4, bias=b.float().to(dev))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_gradient_against_differences(dev):
    lg, dw = logits_of(2, 20, torch.float32).to(dev), randn(2, 4, seed=3).to(dev).double()
    for how in HOWS:
        x = lg.clone().requires_grad_()
        ids, w = moe.route(x, 4, **how)
        d, = torch.autograd.grad(w, x, dw.float())
        step = 2.0 ** -8
        for e in set(ids[1].tolist()) | {0, 11}:
            v = torch.zeros_like(lg)
            v[1, e] = step
            up, down = moe.route(lg + v, 4, **how), moe.route(lg - v, 4, **how)
            assert torch.equal(up[0], ids) and torch.equal(down[0], ids), "choose other inputs"
            diff = ((up[1].double() - down[1].double()) * dw).sum() / (2 * step)
            # step^2 / 6 of a third derivative of at most 6 |g|, and the weights' roundings
            assert abs(diff - d[1, e]) < 2e-4


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("e,groups,top_groups", [(64, 8, 4), (60, 4, 2), (256, 8, 4), (256, 2, 1), (200, 1, 1)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_many_tokens_as_few_at_a_time(dev, dtype, e, groups, top_groups, scores):
    """The lanes that a token has depend on the number of tokens; its experts do not."""
    t = 66000
    lg = logits_of(t, e, dtype).to(dev)
    lg[::1000, : e // 2] = -math.inf
    lg[5::2000] = -math.inf
    lg[7, 3] = math.nan
    for bias in (torch.zeros(e, device=dev), (randn(e, seed=5) * 0.05).to(dev)):
        how = dict(scores=scores, bias=bias, groups=groups, top_groups=top_groups)
        ids, w = moe.route(lg, 8, **how)
        parts = [moe.route(lg[i:i + 3000], 8, **how) for i in range(0, t, 3000)]
        assert torch.equal(ids, torch.cat([p[0] for p in parts]))
        # renormalised weights are of 64-bit scores, to whose factor both sums are the same
        want = torch.cat([p[1] for p in parts])
        assert torch.equal(w.isnan(), want.isnan())
        assert ((w - want).abs() <= 2 * U * want.abs()).logical_or(w.isnan()).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e", [24, 64, 100, 256, 600])
def test_signed_zeros_are_equal(dev, dtype, scores, e):
    g = torch.Generator().manual_seed(e)
    lg = torch.where(torch.rand(40, e, generator=g) < 0.5, -0.0, 0.0).to(dtype)
    lg[20:, ::7] = -1.0
    lg[30:, 5::9] = 1.0
    for bias in (None, torch.zeros(e), -torch.zeros(e)):
        check(dev, lg, 8, scores=scores, bias=bias)
        check(dev, lg, 8, scores=scores, bias=bias, groups=2, top_groups=1)


@pytest.mark.parametrize("how", range(len(HOWS)))
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
def test_biases_that_are_not_finite(dev, how, groups, top_groups):
    """+inf is chosen first, -inf never, NaN last; weights are of the scores alone."""
    t, e = 9, 32
    for value in (math.inf, -math.inf, math.nan):
        bias = randn(e, seed=5) * 0.05
        bias[[3, 9, 30]] = value
        check(dev, logits_of(t, e, torch.float32), 6, randn(t, 6, seed=7), **HOWS[how], bias=bias,
              groups=groups, top_groups=top_groups)
        bias[:] = value
        check(dev, logits_of(t, e, torch.float32), 6, **HOWS[how], bias=bias, groups=groups,
              top_groups=top_groups)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("how", range(len(HOWS)))
@pytest.mark.parametrize("e", [16, 17, 40, 128, 256, 512, 1000])
def test_as_many_slots_as_candidates(dev, dtype, how, e):
    """9 to 16 slots; with keys that are a unit apart, or the same, around the last one."""
    logits = logits_of(25, e, dtype)
    order = logits.float().argsort(-1, descending=True)
    for j in range(8, min(e, 22)):                 # rows 10 to 19: the 9th key on is a cluster
        step = torch.tensor(float(j % 3)) * (2.0 ** -22 if dtype == torch.float32 else 0.0)
        rows = torch.arange(10, 20)
        logits[rows, order[rows, j]] = (logits[rows, order[rows, 8]].float() * (1 - step)).to(dtype)
    logits[20:] = logits[20:, :1]                  # all the same
    for top in (9, 14, 15, 16):
        check(dev, logits, top, randn(25, top, seed=7), **HOWS[how])
        check(dev, logits, top, **HOWS[how], bias=randn(e, seed=5) * 0.05)
        check(dev, logits, top, **HOWS[how], bias=torch.zeros(e))
        if e % 4 == 0 and e // 2 >= top:
            check(dev, logits, top, **HOWS[how], bias=torch.zeros(e), groups=4, top_groups=2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("how", range(len(HOWS)))
@pytest.mark.parametrize("e,groups,top_groups", [
    (9, 1, 1), (23, 1, 1), (33, 3, 2), (60, 4, 2), (65, 5, 3), (72, 8, 4), (100, 1, 1), (130, 1, 1), (144, 12, 4), (257, 1, 1),
    (264, 8, 3), (384, 1, 1), (385, 5, 2), (513, 1, 1), (768, 8, 4), (1023, 1, 1), (1023, 31, 7)])
def test_experts_that_do_not_fill_their_lanes(dev, dtype, how, e, groups, top_groups):
    """Masked, infinite and equal logits where lanes overlap and at the rows' ends."""
    t, top = 21, min(8, e // groups * top_groups)
    logits = logits_of(t, e, dtype)
    logits[3:6, -9:] = 4.0                          # the last ones, all the same
    logits[6:9, -7:] = -math.inf
    logits[9:12, : e - 5] = -math.inf
    logits[12, -1] = logits[13, -8] = math.inf
    logits[14, -2] = math.nan
    logits[15] = logits[15, 0]
    logits[16:18] = -math.inf
    logits[17, -1] = -1.0
    wide = torch.full((t, e + 40), 50.0, dtype=dtype, device=dev)      # what lies beside is higher
    wide[:, 20:e + 20] = logits.to(dev)
    for bias in (None, torch.zeros(e), randn(e, seed=5) * 0.05):
        call = dict(HOWS[how], bias=bias, groups=groups, top_groups=top_groups)
        ids, w = check(dev, logits, top, **call)
        call["bias"] = None if bias is None else bias.to(dev)
        ids2, w2 = moe.route(wide[:, 20:e + 20], top, **call)
        assert torch.equal(ids, ids2) and torch.equal(w.nan_to_num(7.0), w2.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("e,groups,top_groups", [(300, 1, 1), (512, 8, 4), (520, 1, 1), (1000, 20, 4), (1024, 1, 1),
                                                 (1024, 32, 9)])
@pytest.mark.parametrize("how", [0, 1, 2])
def test_many_tokens_of_many_experts(dev, dtype, e, groups, top_groups, how):
    """As a few tokens at a time, which have more lanes."""
    t = 8200
    lg = logits_of(t, e, dtype).to(dev)
    lg[::1000, : e // 2] = -math.inf
    lg[5::2000] = -math.inf
    lg[7, 3] = math.nan
    lg[20:40, ::3] = 2.5
    for top, bias in ((8, None), (15, torch.zeros(e, device=dev)), (16, (randn(e, seed=5) * 0.05).to(dev))):
        call = dict(HOWS[how], bias=bias, groups=groups, top_groups=top_groups)
        ids, w = moe.route(lg, top, **call)
        parts = [moe.route(lg[i:i + 3000], top, **call) for i in range(0, t, 3000)]
        assert torch.equal(ids, torch.cat([p[0] for p in parts]))
        want = torch.cat([p[1] for p in parts])
        assert torch.equal(w.isnan(), want.isnan())
        error = 2 * weight_error(HOWS[how]) + 2 * U
        assert ((w - want).abs() <= error * want.abs()).logical_or(w.isnan()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("how", range(len(HOWS)))
@pytest.mark.parametrize("e", [32, 33, 64, 100, 256, 384, 1000])
def test_seventeen_to_thirty_three_slots(dev, dtype, how, e):
    """With keys that are a unit apart, or the same, around the last one."""
    t = 17
    logits = logits_of(t, e, dtype)
    order = logits.float().argsort(-1, descending=True)
    for j in range(16, min(e, 40)):                # rows 8 to 13: the 17th key on is a cluster
        step = torch.tensor(float(j % 3)) * (2.0 ** -22 if dtype == torch.float32 else 0.0)
        rows = torch.arange(8, 14)
        logits[rows, order[rows, j]] = (logits[rows, order[rows, 16]].float() * (1 - step)).to(dtype)
    logits[14] = logits[14, 0]                     # all the same
    logits[15, 20:] = -math.inf
    logits[16] = -math.inf
    for top in (17, 24, 31, 32) + ((33,) if e > 32 else ()):
        check(dev, logits, top, randn(t, top, seed=7), **HOWS[how])
        check(dev, logits, top, **HOWS[how], bias=randn(e, seed=5) * 0.05)
        check(dev, logits, top, **HOWS[how], bias=torch.zeros(e))
        if e % 4 == 0 and e // 2 >= top:
            check(dev, logits, top, **HOWS[how], bias=torch.zeros(e), groups=4, top_groups=2)
