"""Tokens sorted by expert and back on the device against the 64-bit oracle: the
sort and the copies bit for bit, the sums within the bound of their fp32 terms."""

import pytest
import torch

import oracle.mxfp4 as O
from mx_util import DTYPES, assert_close, big_memory, randn, router  # noqa: F401
from xpu_kernels import moe, mxfp4

pytestmark = pytest.mark.gpu


def routed(t, top, experts, dev, seed=0, dropped=0.0, dtype=torch.int32):
    ids = router(t, top, experts, seed=seed, dropped=dropped, dtype=dtype)
    return ids, moe.sort(ids.to(dev), experts), O.sort(ids, experts)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("t,top,experts,dropped", [
    (1, 1, 1, 0.0), (1, 8, 64, 0.0), (7, 3, 5, 0.3), (64, 1, 2, 0.0), (100, 8, 60, 0.1),
    (1024, 8, 64, 0.0), (1025, 8, 64, 0.05), (3000, 6, 1024, 0.1), (5000, 4, 8, 1.0),
    (20000, 2, 256, 0.02), (2731, 3, 1, 0.5)])
def test_sort(dev, dtype, t, top, experts, dropped):
    _, got, want = routed(t, top, experts, dev, seed=t, dropped=dropped, dtype=dtype)
    for g, w, name in zip(got, want, got._fields):
        assert torch.equal(g.cpu(), w), name


@pytest.mark.parametrize("slots", [63, 64, 65, 1023, 1024, 1025, 2047, 2048, 2049, 4097, 8191,
                                   8192, 8193, 131071, 131072, 131073, 140001])
@pytest.mark.parametrize("experts", [1, 1023, 1024])
def test_sort_sizes(dev, slots, experts):
    _, got, want = routed(slots, 1, experts, dev, seed=slots, dropped=0.03)
    for g, w, name in zip(got, want, got._fields):
        assert torch.equal(g.cpu(), w), name


def test_sort_ids_out_of_range(dev):
    ids = torch.tensor([[0, 1 << 40], [-(1 << 40), 2], [3, 4], [5, 1 << 32], [-1, 4]])
    for i in (ids, ids.clamp(-(1 << 31), (1 << 31) - 1).int()):
        for g, w in zip(moe.sort(i.to(dev), 5), O.sort(i, 5)):
            assert torch.equal(g.cpu(), w)


def test_sort_of_one_expert_and_strided_ids(dev):
    ids = torch.full((3000, 4), 6, dtype=torch.int32)
    for g, w in zip(moe.sort(ids.to(dev), 9), O.sort(ids, 9)):
        assert torch.equal(g.cpu(), w)
    ids = router(50, 8, 16, seed=2).to(dev)[:, ::2]
    for g, w in zip(moe.sort(ids, 16), O.sort(ids, 16)):
        assert torch.equal(g.cpu(), w)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,top,experts,d,dropped", [
    (1, 1, 1, 1, 0.0), (1, 8, 64, 2048, 0.0), (5, 3, 4, 37, 0.4), (33, 2, 8, 512, 0.1),
    (600, 8, 60, 520, 0.05), (2100, 2, 4, 2052, 0.2), (4, 2, 4, 64, 1.0)])
def test_dispatch_and_combine(dev, dtype, t, top, experts, d, dropped):
    _, routing, (oorder, opos, orows, ooff) = routed(t, top, experts, dev, seed=d, dropped=dropped)
    s, live = t * top, int(ooff[-1])
    x = randn(t, d, seed=1, dtype=dtype).to(dev).requires_grad_()
    xs = moe.dispatch(x, routing)
    want = torch.zeros(s, d, dtype=dtype)
    want[:live] = x.detach().cpu()[orows[:live].long()]
    assert torch.equal(xs.cpu(), want)
    dxs = randn(s, d, seed=2, dtype=dtype)
    dxs[live:] = float("nan")                              # rows of no expert are not read
    dx, = torch.autograd.grad(xs, x, dxs.to(dev))
    kept = (opos < live)[..., None]
    rows = torch.where(kept, dxs.double()[opos.long()], 0.0)
    assert_close(dx, rows.sum(1), rows.abs().sum(1), top)

    z = randn(s, d, seed=3, dtype=dtype)
    z[live:] = float("inf")
    zd = z.to(dev).requires_grad_()
    w = torch.rand(t, top, generator=torch.Generator().manual_seed(4))
    w = torch.where(kept[..., 0], w, float("nan"))         # nor are their weights
    wd = w.to(dev).requires_grad_()
    y = moe.combine(zd, routing, wd)
    wz = torch.where(kept, w.double()[..., None] * z.double()[opos.long()], 0.0)
    assert_close(y, wz.sum(1), wz.abs().sum(1), top)
    dy = randn(t, d, seed=5, dtype=dtype)
    dz, dw = torch.autograd.grad(y, (zd, wd), dy.to(dev))
    want = torch.zeros(s, d, dtype=torch.float64)
    want[:live] = w.double().reshape(-1)[oorder[:live].long()][:, None] * dy.double()[orows[:live].long()]
    assert_close(dz, want, want.abs(), 1)
    terms = torch.where(kept, dy.double()[:, None] * z.double()[opos.long()], 0.0)
    assert_close(dw, terms.sum(-1), terms.abs().sum(-1), d)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dev, dtype):
    _, routing, (_, opos, orows, ooff) = routed(30, 3, 8, dev, seed=1)
    base = randn(90, 200, seed=2, dtype=dtype).to(dev)
    w = torch.rand(3, 30, device=dev).t()
    for c in (slice(0, 128), slice(3, 131), slice(1, 2)):
        assert torch.equal(moe.dispatch(base[:30, c], routing), base[:30, c][orows.long()])
        y = moe.combine(base[:, c], routing, w)
        wz = w.cpu().double()[..., None] * base[:, c].cpu().double()[opos.long()]
        assert_close(y, wz.sum(1), wz.abs().sum(1), 3)
    x = base[:30, :64].requires_grad_()
    dx, = torch.autograd.grad(moe.dispatch(x, routing).sum(), x)   # dxs: one value, expanded
    assert (dx == 3).all()


def test_weights_of_another_type(dev):
    _, routing, _ = routed(30, 3, 8, dev, seed=1)
    z = randn(90, 64, seed=2).to(dev)
    w = torch.rand(30, 3, device=dev).bfloat16().requires_grad_()
    y = moe.combine(z, routing, w)
    assert torch.equal(y, moe.combine(z, routing, w.float()))
    y.sum().backward()
    assert w.grad.dtype == torch.bfloat16


def test_gradients_against_differences(dev):
    """Both maps are linear in each argument: the difference quotient is exact up to
    fp32 rounding."""
    _, routing, _ = routed(6, 2, 4, dev, seed=3, dropped=0.2)
    z, w = randn(12, 5, seed=1).to(dev), torch.rand(6, 2, device=dev)
    dy = randn(6, 5, seed=2).to(dev)
    zg, wg = z.clone().requires_grad_(), w.clone().requires_grad_()
    dz, dw = torch.autograd.grad(moe.combine(zg, routing, wg), (zg, wg), dy)

    def loss(z, w):
        return float((moe.combine(z, routing, w).double() * dy.double()).sum())

    for i, j in ((0, 0), (3, 4), (11, 2), (7, 1)):
        step = torch.zeros_like(z)
        step[i, j] = 0.5
        assert abs(loss(z + step, w) - loss(z - step, w) - float(dz[i, j])) < 1e-5
    for i, j in ((0, 0), (2, 1), (5, 0)):
        step = torch.zeros_like(w)
        step[i, j] = 0.5
        assert abs(loss(z, w + step) - loss(z, w - step) - float(dw[i, j])) < 1e-5
    x = randn(6, 5, seed=4).to(dev).requires_grad_()
    dxs = randn(12, 5, seed=5).to(dev)
    dx, = torch.autograd.grad(moe.dispatch(x, routing), x, dxs)
    step = torch.zeros_like(x)
    step[2, 3] = 0.5
    with torch.no_grad():
        rise = ((moe.dispatch(x + step, routing) - moe.dispatch(x - step, routing)) * dxs).sum()
    assert abs(float(rise - dx[2, 3])) < 1e-5


def test_empty(dev):
    routing = moe.sort(torch.empty(0, 2, dtype=torch.int32, device=dev), 4)
    assert routing.offsets.tolist() == [0] * 5 and routing.order.numel() == 0
    x = torch.empty(0, 8, device=dev, requires_grad=True)
    xs = moe.dispatch(x, routing)
    y = moe.combine(xs, routing, torch.empty(0, 2, device=dev))
    assert xs.shape == (0, 8) and y.shape == (0, 8)
    y.sum().backward()
    codes, scales = mxfp4.quantize(randn(4, 8, 32).to(dev))
    x = torch.empty(0, 32, device=dev, requires_grad=True)
    y = mxfp4.grouped_linear(x, codes, scales, routing, gather=True)
    y.sum().backward()
    assert y.shape == (0, 8) and x.grad.shape == (0, 32)


def test_rows_past_4_gib(dev, big_memory):
    t, top, d = 70001, 2, 16384                            # 4.6 GB of sorted rows
    ids = router(t, top, 8, seed=1)
    routing = moe.sort(ids.to(dev), 8)
    x = torch.randn(t, d, dtype=torch.bfloat16, device=dev)
    xs = moe.dispatch(x, routing)
    at = torch.tensor([0, 1, 131071, 131073, t * top - 1], device=dev)
    assert torch.equal(xs[at], x[routing.rows[at].long()])
    w = torch.full((t, top), 0.5, device=dev)
    y = moe.combine(xs, routing, w)                        # a half of the same row twice
    assert torch.equal(y, x)


@pytest.mark.parametrize("t", [1, 5, 150])
def test_ffn(dev, t):
    """The whole path against its steps in 64 bits, the activations rounded and
    quantized where the path does."""
    e, d, f, top = 8, 256, 96, 2
    ids = router(t, top, e, seed=t, dropped=0.1)
    w = torch.rand(t, top, generator=torch.Generator().manual_seed(2))
    x = randn(t, d, seed=1, dtype=torch.bfloat16)
    wu, wd = randn(e, 2 * f, d, seed=3, scale=0.1), randn(e, d, f, seed=4, scale=0.1)
    up, down = mxfp4.quantize(wu.to(dev)), mxfp4.quantize(wd.to(dev))
    xd, wdev = x.to(dev).requires_grad_(), w.to(dev).requires_grad_()
    y = moe.ffn(xd, ids.to(dev), wdev, up, down)
    routing = moe.sort(ids.to(dev), e)
    h = mxfp4.grouped_linear(x.to(dev), *up, routing, gather=True)
    _, opos, orows, ooff = O.sort(ids, e)
    hq = O.dequantize(*O.quantize(x))
    wq = O.dequantize(*O.quantize(wu))
    assert_close(h, O.grouped(hq, wq, orows, ooff), O.grouped(hq.abs(), wq.abs(), orows, ooff), d)
    a = (torch.nn.functional.silu(h[:, :f].float()) * h[:, f:].float()).bfloat16()
    aq, dq = O.dequantize(*O.quantize(a)), O.dequantize(*O.quantize(wd))
    rows = torch.arange(t * top, dtype=torch.int32)
    z = O.grouped(aq, dq, rows, ooff).bfloat16()
    kept = (opos < ooff[-1])[..., None]
    wz = torch.where(kept, w.double()[..., None] * z.double()[opos.long()], 0.0)
    # z's own rounding may differ by an ulp (2^-8) where its fp32 sum does
    got = y.detach().cpu().double()
    assert ((got - wz.sum(1)).abs() <= (2.0 ** -8 + 2.0 ** -9) * wz.abs().sum(1) + 1e-6).all()
    dx, dw = torch.autograd.grad(y, (xd, wdev), torch.ones_like(y))
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all() and (dx != 0).any()
