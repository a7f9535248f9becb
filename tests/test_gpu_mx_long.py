"""More rows and tokens than the threads of one launch."""

import pytest
import torch

import oracle.mxfp4 as O
from mx_util import big_memory  # noqa: F401
from xpu_kernels import moe, mxfp4

pytestmark = pytest.mark.gpu


def test_quantize_and_back(dev, big_memory):
    m = (1 << 28) + 7                                      # 17 GB of rows of one block
    x = torch.empty(m, 32, dtype=torch.bfloat16, device=dev).normal_(generator=torch.Generator(dev).manual_seed(1))
    codes, scales = mxfp4.quantize(x)
    v = mxfp4.dequantize(codes, scales)
    ends = [0, (1 << 26) - 6, (1 << 26) + 1, (1 << 27) - 10, (1 << 28) - 20, m - 5]
    for r in (slice(a, a + 5) for a in ends):
        oc, os_ = O.quantize(x[r])
        assert torch.equal(codes[r].cpu(), oc) and torch.equal(scales[r].cpu(), os_)
        assert torch.equal(v[r].cpu(), O.dequantize(oc, os_).to(torch.bfloat16))
    # every value is within its block's largest step, a quarter of the maximum's binade
    for a in range(0, m, 1 << 25):
        part = x[a:a + (1 << 25)].float()
        assert ((v[a:a + (1 << 25)].float() - part).abs().amax(-1) <= part.abs().amax(-1) * 0.25).all()


def test_routing(dev, big_memory):
    t, e, d = (1 << 26) + 9, 3, 8
    g = torch.Generator(dev).manual_seed(2)
    ids = torch.randint(-1, e, (t, 1), generator=g, device=dev, dtype=torch.int32)
    routing = moe.sort(ids, e)
    key = torch.where(ids[:, 0] < 0, e, ids[:, 0])
    order = torch.sort(key, stable=True).indices
    assert torch.equal(routing.order.long(), order)
    live = int((ids >= 0).sum())
    assert int(routing.offsets[-1]) == live
    x = torch.empty(t, d, dtype=torch.bfloat16, device=dev).normal_(generator=g).requires_grad_()
    xs = moe.dispatch(x, routing)
    assert torch.equal(xs[:live], x[order[:live]]) and not xs[live:].any()
    z = xs.detach().clone().requires_grad_()
    w = torch.rand(t, 1, generator=g, device=dev).requires_grad_()
    y = moe.combine(z, routing, w)
    kept = ids >= 0
    want = torch.where(kept, w * x.detach().float(), 0.0).bfloat16()
    assert torch.equal(y, want)
    del want
    dx, = torch.autograd.grad(xs, x, z.detach())
    assert torch.equal(dx, torch.where(kept, x, 0).detach())
    dy = torch.empty(t, d, dtype=torch.bfloat16, device=dev).normal_(generator=g)
    dz, dw = torch.autograd.grad(y, (z, w), dy)
    assert torch.equal(dz[:live], (w.detach() * dy.float()).bfloat16()[order[:live]]) and not dz[live:].any()
    # eight products, fp32 sums in either order
    terms = dy.float() * x.detach().float()
    bound = 8 * 2.0 ** -23 * terms.abs().sum(-1, keepdim=True)
    assert ((dw - torch.where(kept, terms.sum(-1, keepdim=True), 0.0)).abs() <= bound).all()
