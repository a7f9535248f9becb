"""The experts' operators put together: wrong routings refused alike with and without the
native host path, the gradients of the whole FFN step by step against 64 bits, and
captured steps with their gradients."""

import pytest
import torch

import oracle.mxfp4 as O
from mx_util import DTYPES, HALF_ULP, assert_close, randn, router
from xpu_kernels import int8, moe, mxfp4
from xpu_kernels.int8 import _lib as L

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ refusals
def outcome(fn):
    try:
        r = fn()
    except Exception as e:
        assert "argument" not in str(e), f"the call itself is wrong: {e}"
        return type(e).__name__, str(e)
    return [r] if isinstance(r, torch.Tensor) else list(r)


@pytest.mark.parametrize("t", [2, 30, 300])
def test_combine_of_wrong_routings(dev, monkeypatch, t):
    """The same refusal, or the same result, through both host paths."""
    top, experts, d = 3, 6, 288
    ids = router(t, top, experts, seed=t, dropped=0.1).to(dev)
    routing = moe.sort(ids, experts)
    z = randn(t * top, d, seed=1, dtype=torch.bfloat16).to(dev)
    w = torch.rand(t, top, device=dev)
    long, one = moe.Routing(*(q.long() for q in routing)), moe.sort(ids[:, :1], experts)
    cases = {
        "right": (z, routing, w, None),
        "other experts": (z, moe.sort(ids, experts - 1), w, None),
        "tuple": (z, tuple(routing), w, TypeError), "none": (z, None, w, TypeError),
        "cpu": (z, moe.Routing(*(q.cpu() for q in routing)), w, TypeError),
        "long": (z, long, w, TypeError), "long position": (z, routing._replace(position=long.position), w, TypeError),
        "strided": (z, routing._replace(order=torch.stack([routing.order] * 2, 1)[:, 0]), w, TypeError),
        "fewer tokens": (z, moe.sort(ids[1:], experts), w, ValueError),
        "one slot": (z, one, w, ValueError), "mixed": (z, routing._replace(position=one.position), w, ValueError),
        "no offsets": (z, routing._replace(offsets=routing.offsets[:1]), w, ValueError),
        "flat position": (z, routing._replace(position=routing.position.reshape(-1)), w, ValueError),
        "rows missing": (z[1:], routing, w, ValueError), "z of one dimension": (z[:, 0], routing, w, ValueError),
        "weights' shape": (z, routing, w.t(), ValueError), "weights on the cpu": (z, routing, w.cpu(), TypeError),
        "no weights": (z, routing, None, TypeError), "weights of whole numbers": (z, routing, w.int(), TypeError),
    }
    for name, (z_, r, w_, error) in cases.items():
        fast = outcome(lambda: moe.combine(z_, r, w_))
        with monkeypatch.context() as m:
            m.setattr(L, "HOST", None)
            slow = outcome(lambda: moe.combine(z_, r, w_))
        if error is None:
            assert isinstance(fast, list) and torch.equal(fast[0], slow[0]), name
        else:
            assert fast == slow and fast[0] == error.__name__, (name, fast, slow)


@pytest.mark.parametrize("top,experts", [(3, 6)])
def test_no_expert_for_any_slot(dev, top, experts):
    """Rows whose mask leaves nothing: zeros, and no gradient."""
    t, d, f = 20, 64, 32
    ids = torch.full((t, top), -1, dtype=torch.int64, device=dev)
    up = mxfp4.quantize(randn(experts, 2 * f, d, seed=1).to(dev))
    down = mxfp4.quantize(randn(experts, d, f, seed=2).to(dev))
    x = randn(t, d, seed=3, dtype=torch.bfloat16).to(dev).requires_grad_()
    w = torch.rand(t, top, device=dev).requires_grad_()
    y = moe.ffn(x, ids, w, up, down)
    dx, dw = torch.autograd.grad(y, (x, w), torch.full_like(y, float("nan")))
    assert not y.any() and not dx.any() and not dw.any()


# ----------------------------------------------------------------- the FFN
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,dropped", [(1, 0.0), (5, 0.3), (150, 0.1)])
def test_ffn_gradients(dev, dtype, t, dropped):
    """The FFN's gradients are bit for bit those of its steps, and each step's are within
    the bound of its fp32 sums and one rounding of the formula in 64 bits."""
    e, d, f, top = 8, 256, 96, 2
    ids = router(t, top, e, seed=t, dropped=dropped)
    _, opos, orows, ooff = O.sort(ids, e)
    wu, wd = randn(e, 2 * f, d, seed=3, scale=0.1), randn(e, d, f, seed=4, scale=0.1)
    up, down = mxfp4.quantize(wu.to(dev)), mxfp4.quantize(wd.to(dev))
    uq, dq = O.dequantize(*O.quantize(wu)), O.dequantize(*O.quantize(wd))
    x = randn(t, d, seed=1, dtype=dtype).to(dev).requires_grad_()
    w = torch.rand(t, top, generator=torch.Generator().manual_seed(2)).to(dev).requires_grad_()
    dy = randn(t, d, seed=5, dtype=dtype).to(dev)
    y = moe.ffn(x, ids.to(dev), w, up, down)
    dx, dw = torch.autograd.grad(y, (x, w), dy)

    routing = moe.sort(ids.to(dev), e)
    leaf = x.detach().clone().requires_grad_()
    h = mxfp4.grouped_linear(leaf, *up, routing, gather=True)
    hl = h.detach().clone().requires_grad_()
    gate, value = hl.chunk(2, dim=-1)
    a = (torch.nn.functional.silu(gate.float()) * value.float()).to(dtype)
    al = a.detach().clone().requires_grad_()
    z = mxfp4.grouped_linear(al, *down, routing)
    zl, wl = z.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    dz, dw2 = torch.autograd.grad(moe.combine(zl, routing, wl), (zl, wl), dy)
    da, = torch.autograd.grad(z, al, dz)
    dh, = torch.autograd.grad(a, hl, da)
    dx2, = torch.autograd.grad(h, leaf, dh)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)

    r = t * top
    every = torch.arange(r, dtype=torch.int32)
    kept = (opos < ooff[-1])[..., None]
    live = int(ooff[-1])
    g64 = dy.cpu().double()
    w64 = torch.zeros(r, 1, dtype=torch.float64)
    w64[opos.reshape(-1).long(), 0] = w.detach().cpu().double().reshape(-1)
    want = w64 * g64[orows.long()]
    want[live:] = 0
    assert_close(dz, want, want.abs(), 1)
    terms = torch.where(kept, g64[:, None] * z.detach().cpu().double()[opos.long()], 0.0)
    assert_close(dw, terms.sum(-1), terms.abs().sum(-1), d)
    z64, down_t, up_t = dz.cpu().double(), dq.transpose(1, 2), uq.transpose(1, 2)
    assert_close(da, O.grouped(z64, down_t, every, ooff), O.grouped(z64.abs(), down_t.abs(), every, ooff), 3 * d)
    # silu(g) v: fp32 steps of a relative 2^-23 each, sixteen at most, on terms of these sizes
    a64, gate, value = da.cpu().double(), h.detach().cpu().double()[:, :f], h.detach().cpu().double()[:, f:]
    s = torch.sigmoid(gate)
    want = torch.cat([a64 * value * s * (1 + gate * (1 - s)), a64 * gate * s], 1)
    size = torch.cat([(a64 * value).abs() * (1 + gate.abs()), (a64 * gate).abs()], 1)
    bound = 2.0 ** -19 * size + HALF_ULP[dtype] * (want.abs() + 2.0 ** -19 * size) + 1e-7 * (dtype == torch.float16)
    assert ((dh.cpu().double() - want).abs() <= bound).all()
    h64 = dh.cpu().double()
    dxs, mag = O.grouped(h64, up_t, every, ooff), O.grouped(h64.abs(), up_t.abs(), every, ooff)
    assert_close(dx, dxs[opos.long()].sum(1), mag[opos.long()].sum(1), 3 * 2 * f + top)
    assert dx.any() and dw.any()


@pytest.mark.parametrize("n", [16, 512, 2064])
def test_bias_gradient_is_the_int8_linears(dev, n):
    """bf16 sums of a bf16 dy: bit for bit int8.column_sum's."""
    dy = randn(1025, n, seed=n, dtype=torch.bfloat16).to(dev)
    codes, scales = mxfp4.quantize(randn(n, 32, seed=3).to(dev))
    b = torch.zeros(n, dtype=torch.bfloat16, device=dev, requires_grad=True)
    y = mxfp4.linear(torch.ones(1025, 32, dtype=torch.bfloat16, device=dev), codes, scales, b)
    assert torch.equal(torch.autograd.grad(y, b, dy)[0], int8.column_sum(dy))


# -------------------------------------------------------------------- graphs
def replays(step, refresh):
    """step() captured, replayed after refresh(seed) and compared with itself run eagerly."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (5, 6, 7, 8):
        refresh(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in out]
        for g, w in zip(got, step()):
            assert torch.equal(g, w)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,top,e", [(4, 2, 8), (700, 3, 16), (3000, 4, 16)])
def test_routing_in_a_graph(dev, dtype, t, top, e):
    d = 264
    ids = router(t, top, e, seed=3).to(dev)
    x = randn(t, d, seed=1, dtype=dtype).to(dev).requires_grad_()
    w = torch.rand(t, top, device=dev).requires_grad_()
    dy = randn(t, d, seed=2, dtype=dtype).to(dev)

    def step():
        routing = moe.sort(ids, e)
        y = moe.combine(moe.dispatch(x, routing), routing, w)
        return (*routing, y, *torch.autograd.grad(y, (x, w), dy))

    def refresh(seed):
        ids.copy_(router(t, top, e, seed=seed, dropped=0.1))
        with torch.no_grad():
            x.copy_(randn(t, d, seed=seed, dtype=dtype))
            w.copy_(torch.rand(t, top, generator=torch.Generator().manual_seed(seed)))
        dy.copy_(randn(t, d, seed=seed + 9, dtype=dtype))

    replays(step, refresh)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,top,e", [(4, 2, 8), (700, 3, 8)])
def test_ffn_in_a_graph(dev, dtype, t, top, e):
    d, f = 288, 160
    up = mxfp4.quantize(randn(e, 2 * f, d, seed=3, scale=0.1).to(dev))
    down = mxfp4.quantize(randn(e, d, f, seed=4, scale=0.1).to(dev))
    ids = router(t, top, e, seed=3).to(dev)
    x = randn(t, d, seed=1, dtype=dtype).to(dev).requires_grad_()
    w = torch.rand(t, top, device=dev).requires_grad_()
    dy = randn(t, d, seed=2, dtype=dtype).to(dev)

    def step():
        y = moe.ffn(x, ids, w, up, down)
        return (y, *torch.autograd.grad(y, (x, w), dy))

    def refresh(seed):
        ids.copy_(router(t, top, e, seed=seed, dropped=0.1))
        with torch.no_grad():
            x.copy_(randn(t, d, seed=seed, dtype=dtype))
        dy.copy_(randn(t, d, seed=seed + 9, dtype=dtype))

    replays(step, refresh)
