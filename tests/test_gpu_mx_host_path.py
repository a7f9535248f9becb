"""The MXFP4 and routing calls through the native host path and without it: the same
tensors, bit for bit, or the same error."""

import pytest
import torch

from mx_util import randn, router
from xpu_kernels import moe, mxfp4
from xpu_kernels.int8 import _lib as L

pytestmark = pytest.mark.gpu


def outcome(fn):
    try:
        r = fn()
    except Exception as e:
        return type(e).__name__, str(e)
    return [r] if isinstance(r, torch.Tensor) else list(r)


def both(monkeypatch, fn, name):
    assert L.HOST is not None
    fast = outcome(fn)
    with monkeypatch.context() as m:
        m.setattr(L, "HOST", None)
        slow = outcome(fn)
    assert type(fast) is type(slow), (name, fast, slow)
    if isinstance(fast, tuple):
        assert fast == slow, name
        return False
    for a, b in zip(fast, slow):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride(), name
        assert torch.equal(a.detach().view(torch.uint8), b.detach().view(torch.uint8)), name
    return True


def forms(dev, m, k, dtype=torch.bfloat16):
    x = randn(m, k, seed=1, dtype=dtype).to(dev)
    wide = randn(m + 3, 2 * k, seed=2, dtype=dtype).to(dev)
    return {"plain": x, "batched": x.reshape(1, m, k), "vector": x[0], "columns": wide[:m, :k],
            "misaligned": wide[3:, 1:k + 1], "transposed": randn(k, m, seed=3, dtype=dtype).to(dev).t(),
            "expanded": x[:1].expand(m, k), "fp32": x.float(), "fp16": x.half(), "double": x.double(),
            "cpu": x.cpu(), "empty": x[:0], "short": x[:, :k - 8].contiguous(), "int": x.int(),
            "scalar": x[0, 0], "grad": x.clone().requires_grad_(), "not a tensor": 3}


@pytest.mark.parametrize("m", [3, 40, 150])
def test_quantize_and_linear(dev, monkeypatch, m):
    k, n = 544, 72
    codes, scales = mxfp4.quantize(randn(n, k, seed=5).to(dev))
    answered = 0
    for name, x in forms(dev, m, k).items():
        answered += both(monkeypatch, lambda: mxfp4.quantize(x), name)
        answered += both(monkeypatch, lambda: mxfp4.linear(x, codes, scales), name)
    assert answered >= 20
    x = randn(m, k, seed=1, dtype=torch.bfloat16).to(dev)
    b = randn(2 * n, seed=6).to(dev)
    for name, bias in {"fp32": b[:n], "bf16": b[:n].bfloat16(), "fp16": b[:n].half(), "strided": b[::2],
                       "row": b[:n].reshape(1, n), "wrong": b, "cpu": b[:n].cpu(), "int": b[:n].int(),
                       "grad": b[:n].clone().requires_grad_(), "not a tensor": 1.0}.items():
        both(monkeypatch, lambda: mxfp4.linear(x, codes, scales, bias), name)
    for name, (c, s) in {"row slice": (codes[8:], scales[8:]), "columns": (codes[:, ::2], scales),
                         "int8": (codes.view(torch.int8), scales), "unpadded": (codes, scales[:, :17]),
                         "cpu": (codes.cpu(), scales), "batched": (codes[None], scales[None]),
                         "fewer scales": (codes, scales[1:])}.items():
        both(monkeypatch, lambda: mxfp4.linear(x, c, s), name)
        both(monkeypatch, lambda: mxfp4.dequantize(c, s), name)
        both(monkeypatch, lambda: mxfp4.dequantize(c, s, torch.int32), name)


@pytest.mark.parametrize("t", [2, 30, 300])
def test_experts(dev, monkeypatch, t):
    top, experts, k, n = 3, 6, 288, 40
    ids = router(t, top, experts, seed=t, dropped=0.1).to(dev)
    for name, i in {"int32": ids, "int64": ids.long(), "strided": ids.t().contiguous().t(), "int16": ids.short(),
                    "cpu": ids.cpu(), "flat": ids.reshape(-1), "empty": ids[:0], "none": None}.items():
        both(monkeypatch, lambda: moe.sort(i, experts), name)
    for e in (0, 1, 1024, 1025, 2.0, "6"):
        both(monkeypatch, lambda: moe.sort(ids, e), str(e))
    routing = moe.sort(ids, experts)
    codes, scales = mxfp4.quantize(randn(experts, n, k, seed=5).to(dev))
    answered = 0
    for name, x in forms(dev, t, k).items():
        answered += both(monkeypatch, lambda: moe.dispatch(x, routing), name)
        answered += both(monkeypatch, lambda: mxfp4.grouped_linear(x, codes, scales, routing, gather=True), name)
    w = torch.rand(t, top, device=dev)
    for name, z in forms(dev, t * top, k).items():
        answered += both(monkeypatch, lambda: moe.combine(z, routing), name)
        answered += both(monkeypatch, lambda: moe.combine(z, routing, w), name)
        answered += both(monkeypatch, lambda: mxfp4.grouped_linear(z, codes, scales, routing), name)
    assert answered >= 30
    z = randn(t * top, k, seed=1, dtype=torch.bfloat16).to(dev)
    for name, v in {"bf16": w.bfloat16(), "strided": torch.rand(top, t, device=dev).t(), "flat": w.reshape(-1),
                    "cpu": w.cpu(), "int": w.int(), "grad": w.clone().requires_grad_()}.items():
        both(monkeypatch, lambda: moe.combine(z, routing, v), name)
    for name, r in {"tuple": tuple(routing), "cpu": moe.Routing(*(q.cpu() for q in routing)),
                    "other": moe.sort(ids[1:], experts), "long": moe.Routing(*(q.long() for q in routing)),
                    "fewer experts": moe.sort(ids, experts - 1)}.items():
        both(monkeypatch, lambda: moe.dispatch(z[:t], r), name)
        both(monkeypatch, lambda: moe.combine(z, r), name)
        both(monkeypatch, lambda: mxfp4.grouped_linear(z, codes, scales, r), name)


def dys(dev, m, n, dtype=torch.bfloat16):
    base = randn(m + 2, n + 16, seed=8, dtype=dtype).to(dev)
    return {"plain": base[:m, :n].contiguous(), "columns": base[:m, :n], "misaligned": base[1:m + 1, 3:n + 3],
            "expanded": base[:1, :n].expand(m, n), "one value": base[:1, :1].expand(m, n)}


@pytest.mark.parametrize("m", [3, 150])
def test_gradients(dev, monkeypatch, m):
    k, n, top, experts = 288, 48, 3, 6
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        codes, scales = mxfp4.quantize(randn(n, k, seed=5).to(dev))
        x = randn(m, k, seed=1, dtype=dtype).to(dev).requires_grad_()
        b = randn(n, seed=6).to(dev).requires_grad_()
        for name, dy in dys(dev, m, n, dtype).items():
            assert both(monkeypatch, lambda: torch.autograd.grad(mxfp4.linear(x, codes, scales, b), (x, b), dy), name)
            assert both(monkeypatch, lambda: torch.autograd.grad(
                mxfp4.linear(x[None], codes, scales), x, dy[None]), name)
        codes, scales = mxfp4.quantize(randn(experts, n, k, seed=5).to(dev))
        routing = moe.sort(router(m, top, experts, seed=m, dropped=0.1).to(dev), experts)
        w = torch.rand(m, top, device=dev).requires_grad_()
        z = randn(m * top, k, seed=2, dtype=dtype).to(dev).requires_grad_()
        for gather, xs in ((True, x), (False, z)):
            for name, dy in dys(dev, m * top, n, dtype).items():
                assert both(monkeypatch, lambda: torch.autograd.grad(
                    mxfp4.grouped_linear(xs, codes, scales, routing, gather=gather), xs, dy), name)
        for name, dy in dys(dev, m * top, k, dtype).items():
            assert both(monkeypatch, lambda: torch.autograd.grad(moe.dispatch(x, routing), x, dy), name)
        for name, dy in dys(dev, m, k, dtype).items():
            assert both(monkeypatch, lambda: torch.autograd.grad(moe.combine(z, routing, w), (z, w), dy), name)


def test_second_derivatives_are_refused(dev):
    codes, scales = mxfp4.quantize(randn(48, 288, seed=5).to(dev))
    x = randn(9, 288, seed=1, dtype=torch.bfloat16).to(dev).requires_grad_()
    dy = randn(9, 48, seed=2, dtype=torch.bfloat16).to(dev).requires_grad_()
    dx, = torch.autograd.grad(mxfp4.linear(x, codes, scales), x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()
