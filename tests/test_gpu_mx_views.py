"""Lazily negated tensors and batched gradients."""

import pytest
import torch

from mx_util import randn, router
from xpu_kernels import moe, mxfp4
from xpu_kernels.int8 import _lib as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
def test_lazily_negated_tensors(dev, monkeypatch, native):
    """A tensor whose sign is a flag of its view (torch's imaginary part of a conjugate)
    counts with that sign, in every argument and as a gradient."""
    if not native:
        monkeypatch.setattr(L, "HOST", None)
    neg = torch._neg_view
    t, top, e, k, n = 40, 2, 4, 96, 48
    codes, scales = mxfp4.quantize(randn(n, k, seed=1).to(dev))
    ws, ss = mxfp4.quantize(randn(e, n, k, seed=2).to(dev))
    routing = moe.sort(router(t, top, e, seed=3, dropped=0.1).to(dev), e)
    x, z = randn(t, k, seed=4).to(dev), randn(t * top, k, seed=5).to(dev)
    b, w = randn(n, seed=6).to(dev), torch.rand(t, top, device=dev)
    for call in (lambda f: mxfp4.quantize(f(x))[0], lambda f: mxfp4.linear(f(x), codes, scales, b),
                 lambda f: mxfp4.linear(x, codes, scales, f(b)),
                 lambda f: mxfp4.grouped_linear(f(z), ws, ss, routing),
                 lambda f: mxfp4.grouped_linear(f(x), ws, ss, routing, gather=True),
                 lambda f: moe.dispatch(f(x), routing), lambda f: moe.combine(f(z), routing, w),
                 lambda f: moe.combine(z, routing, f(w))):
        assert torch.equal(call(neg), call(torch.neg))
    xg, zg, bg, wg = (v.clone().requires_grad_() for v in (x, z, b, w))
    dy, dk = randn(t, n, seed=7).to(dev), randn(t, k, seed=8).to(dev)
    dz, dzn = randn(t * top, k, seed=9).to(dev), randn(t * top, n, seed=10).to(dev)
    for out, into, g in ((mxfp4.linear(xg, codes, scales, bg), (xg, bg), dy),
                         (mxfp4.grouped_linear(xg, ws, ss, routing, gather=True), (xg,), dzn),
                         (mxfp4.grouped_linear(zg, ws, ss, routing), (zg,), dzn),
                         (moe.dispatch(xg, routing), (xg,), dz), (moe.combine(zg, routing, wg), (zg, wg), dk)):
        for a, c in zip(torch.autograd.grad(out, into, neg(g), retain_graph=True),
                        torch.autograd.grad(out, into, -g)):
            assert torch.equal(a, c)


@pytest.mark.parametrize("native", [True, False])
def test_batched_gradients_are_refused(dev, monkeypatch, native):
    if not native:
        monkeypatch.setattr(L, "HOST", None)
    codes, scales = mxfp4.quantize(randn(48, 96, seed=1).to(dev))
    x = randn(8, 96, seed=4).to(dev).requires_grad_()
    y = mxfp4.linear(x, codes, scales)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, x, randn(3, 8, 48, seed=2).to(dev), is_grads_batched=True)
