"""RMS norm, routing and rotary positions through the native host path and without it: the
same tensors in the same layout, bit for bit, the same gradients, or the same error."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from mx_util import randn
from test_gpu_mx_host_path import forms, outcome
from xpu_kernels import moe, norm, rope
from xpu_kernels.int8 import _lib as L

pytestmark = pytest.mark.gpu


def both(monkeypatch, fn, name):
    """Whether fn has results, the same ones with the native host path and without."""
    assert L.HOST is not None
    fast = outcome(fn)
    with monkeypatch.context() as m:
        m.setattr(L, "HOST", None)
        slow = outcome(fn)
    assert type(fast) is type(slow), (name, fast, slow)
    if isinstance(fast, tuple):
        assert fast == slow, name
        return False
    assert len(fast) == len(slow), name
    for a, b in zip(fast, slow):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride(), name
        a, b = (t.detach().contiguous().reshape(-1).view(torch.uint8) for t in (a, b))
        assert torch.equal(a, b), name
    return True


def test_norm(dev, monkeypatch):
    k = 512
    w, answered = randn(k, seed=5).to(dev), 0
    for name, x in forms(dev, 6, k).items():
        for r in (None, x, randn(6, k, seed=7, dtype=torch.bfloat16).to(dev), 1.0):
            answered += both(monkeypatch, lambda: norm.rms_norm(x, None, 1e-5, residual=r), name)
            answered += both(monkeypatch, lambda: norm.rms_norm_int8(x, None, 1e-5, residual=r), name)
        answered += both(monkeypatch, lambda: norm.rms_norm(x, w), name)
    assert answered >= 40
    x = randn(6, k, seed=1, dtype=torch.float16).to(dev)
    for name, v in {"fp16": w.half(), "bf16": w.bfloat16(), "strided": randn(2 * k, seed=6).to(dev)[::2],
                    "row": w[None], "long": randn(k + 8, seed=1).to(dev), "cpu": w.cpu(), "int": w.int(),
                    "grad": w.clone().requires_grad_(), "not a tensor": 2.0}.items():
        both(monkeypatch, lambda: norm.rms_norm(x, v), name)
        both(monkeypatch, lambda: norm.rms_norm_int8(x, v, rotate=False), name)
    for eps in (0, 0.0, 1, -1.0, float("nan"), float("inf"), "1", None, 1 << 2000, True):
        both(monkeypatch, lambda: norm.rms_norm(x, w, eps), str(eps)[:20])
    for rotate in (True, False, 0, 1, "yes", None):
        both(monkeypatch, lambda: norm.rms_norm_int8(x[:, :300], None, rotate=rotate), str(rotate))
        both(monkeypatch, lambda: norm.rms_norm_int8(x, None, rotate=rotate), str(rotate))


def test_route(dev, monkeypatch):
    answered = 0
    for name, x in forms(dev, 9, 64).items():
        for how in (dict(), dict(scores="sigmoid", groups=8, top_groups=3), dict(renormalize=False, scale=2)):
            answered += both(monkeypatch, lambda: moe.route(x, 4, **how), name)
    assert answered >= 20
    x, b = randn(9, 64, seed=1).to(dev), randn(128, seed=2).to(dev)
    for name, how in {"bias": dict(bias=b[:64]), "strided": dict(bias=b[::2]), "bf16": dict(bias=b[:64].bfloat16()),
                      "long": dict(bias=b), "cpu": dict(bias=b[:64].cpu()), "one": dict(bias=1.0),
                      "grad": dict(bias=b[:64].clone().requires_grad_()), "scores": dict(scores="tanh"),
                      "no scores": dict(scores=None), "groups": dict(groups=7), "zero": dict(groups=0),
                      "top groups": dict(groups=4, top_groups=5), "few": dict(groups=32, top_groups=1),
                      "float": dict(groups=4.0), "true": dict(top_groups=True), "scale": dict(scale="2"),
                      "huge": dict(scale=1e300), "none": dict(scale=None)}.items():
        both(monkeypatch, lambda: moe.route(x, 4, **how), name)
    for top in (0, 1, 64, 65, -1, 2.0, None, 1 << 70, True):
        both(monkeypatch, lambda: moe.route(x, top), str(top))
    both(monkeypatch, lambda: moe.route(randn(2, 1025, seed=1).to(dev), 2), "experts")


def test_rotate_axes(dev, monkeypatch):
    b, s, h, d = 2, 5, 4, 32
    f = rope.axis_frequencies((6, 4, 3), device=dev)
    p = torch.randint(0, 99, (3, b, s), dtype=torch.int32, device=dev)
    q = randn(b, s, h, d, seed=1).to(dev)
    wide = randn(b, s, 3 * h * d + 1, seed=2).to(dev)
    base = randn(b, h, s, d, seed=3).to(dev)
    heads = {"plain": q, "bf16": q.bfloat16(), "fp16": q.half(), "columns": wide[..., 1:h * d + 1].unflatten(-1, (h, d)),
             "heads first": base.transpose(1, 2), "every other": base.transpose(1, 2)[:, :, ::2],
             "expanded": base[:, :1].transpose(1, 2).expand(b, s, h, d), "reversed": q.transpose(2, 3).contiguous().transpose(2, 3),
             "one": q[:, :, :1, :], "grad": q.clone().requires_grad_(), "double": q.double(), "cpu": q.cpu(),
             "flat": q.flatten(2), "empty": q[:, :0], "short": q[..., :8], "other": q[:1], "no": 3,
             "negated": torch._neg_view(q), "no heads": q[:, :, :0]}
    answered = 0
    for name, x in heads.items():
        for other in (None, x, q, q[:, :, :1].bfloat16()):
            for split in (True, False):
                answered += both(monkeypatch, lambda: [
                    t for t in rope.rotate_axes(x, other, p, f, split_half=split) if t is not None], name)
    assert answered >= 60
    for name, pos in {"int64": p.long(), "fp32": p.float(), "of all": p[:, 0], "strided": p.transpose(1, 2).contiguous().transpose(1, 2),
                      "expanded": p[:1].expand(3, b, s), "one axis": p[:1], "int16": p.short(), "cpu": p.cpu(),
                      "flat": p[0, 0], "short": p[..., :4], "double": p.double(), "list": [1],
                      "grad": p.float().requires_grad_(), "17": p[:1].expand(17, b, s), "none": p[:0]}.items():
        both(monkeypatch, lambda: rope.rotate_axes(q, q, pos, f), name)
    F = rope.AxisFrequencies
    for name, g in {"tuple": tuple(f), "fp32": F(f.inv_freq.float(), f.axis), "int64": F(f.inv_freq, f.axis.long()),
                    "short": F(f.inv_freq[:9], f.axis), "cpu": F(f.inv_freq.cpu(), f.axis), "none": F(None, f.axis),
                    "strided": F(f.inv_freq.repeat(2)[::2], f.axis), "empty": F(f.inv_freq[:0], f.axis[:0]),
                    "many": rope.axis_frequencies((17,), device=dev), "offset": F(f.inv_freq[1:], f.axis[1:])}.items():
        both(monkeypatch, lambda: rope.rotate_axes(q, q, p, g), name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients(dev, monkeypatch, dtype):
    """Each combination of inputs that need one and outputs that have one."""
    b, s, h, d = 2, 5, 4, 32
    f = rope.axis_frequencies((6, 4, 3), device=dev)
    p = torch.randint(0, 99, (3, b, s), dtype=torch.int32, device=dev)
    x, r, w = (randn(6, 320, seed=i, dtype=dtype).to(dev) for i in (1, 2, 3))
    w, lg = w[0].float().clone(), randn(7, 64, seed=4, dtype=dtype).to(dev)
    q, k = randn(b, s, h, d, seed=5, dtype=dtype).to(dev), randn(b, s, 1, d, seed=6, dtype=dtype).to(dev)

    def grads(fn, tensors, mask, outputs):
        leaves = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(tensors)]
        out = fn(*leaves)
        out = [t for t in (out if isinstance(out, tuple) else (out,)) if t is not None and t.is_floating_point()]
        into = [t for t in leaves if t.requires_grad]
        picked = [t for i, t in enumerate(out) if outputs >> i & 1 and t.requires_grad]
        if not picked or not into:
            return out
        g = torch.autograd.grad(picked, into, [randn(*t.shape, seed=9 + i, dtype=t.dtype).to(dev)
                                               for i, t in enumerate(picked)], allow_unused=True)
        return out + [t if t is not None else torch.zeros(1, device=dev) for t in g]

    for mask in range(1, 8):
        for outputs in (1, 2, 3):
            for name, fn, tensors in (
                    ("norm", lambda a, c: norm.rms_norm(a, c), (x, w)),
                    ("norm, no weight", lambda a, c: norm.rms_norm(a, residual=c), (x, r)),
                    ("norm, residual", lambda a, c, e: norm.rms_norm(a, c, residual=e), (x, w, r)),
                    ("route", lambda a: moe.route(a, 4)[1], (lg,)),
                    ("route, groups", lambda a: moe.route(a, 4, scores="sigmoid", groups=4, top_groups=2)[1], (lg,)),
                    ("rope", lambda a, c: rope.rotate_axes(a, c, p, f), (q, k)),
                    ("rope, q", lambda a: rope.rotate_axes(a, None, p, f), (q,))):
                both(monkeypatch, lambda: grads(fn, tensors, mask, outputs), name)


@pytest.mark.parametrize("native", [True, False])
def test_refused_derivatives(dev, monkeypatch, native):
    """Forward mode, second and batched derivatives."""
    if not native:
        monkeypatch.setattr(L, "HOST", None)
    f = rope.axis_frequencies((8,), device=dev)
    p = torch.arange(3, device=dev)[None]
    x, w, lg = randn(4, 64, seed=1).to(dev), randn(64, seed=2).to(dev), randn(4, 16, seed=3).to(dev)
    q = randn(1, 3, 2, 16, seed=4).to(dev)
    calls = [(x, lambda v: norm.rms_norm(v, w)), (w, lambda v: norm.rms_norm(x, v)),
             (x, lambda v: norm.rms_norm(x, w, residual=v)[0]), (x, lambda v: norm.rms_norm_int8(v, rotate=False)),
             (lg, lambda v: moe.route(v, 2)[1]), (q, lambda v: rope.rotate_axes(v, None, p, f)[0]),
             (q, lambda v: rope.rotate_axes(q, v, p, f)[1])]
    for v, call in calls:
        with fwad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(fwad.make_dual(v, torch.ones_like(v)))
        a = v.clone().requires_grad_()
        try:
            y = call(a)
        except RuntimeError as e:
            assert "no gradient" in str(e)
            continue
        with pytest.raises(RuntimeError):
            g, = torch.autograd.grad(y, a, torch.ones_like(y).requires_grad_(), create_graph=True)
            g.sum().backward()
        with pytest.raises(RuntimeError):
            y = call(a)
            torch.autograd.grad(y, a, torch.ones(3, *y.shape, device=dev), is_grads_batched=True)


@pytest.mark.parametrize("native", [True, False])
def test_lazily_negated(dev, monkeypatch, native):
    if not native:
        monkeypatch.setattr(L, "HOST", None)
    neg = torch._neg_view
    f = rope.axis_frequencies((8,), device=dev)
    p = torch.arange(3, device=dev)[None]
    x, w, lg = randn(4, 64, seed=1).to(dev), randn(64, seed=2).to(dev), randn(4, 64, seed=3).to(dev)
    q = randn(1, 3, 2, 16, seed=4).to(dev)
    for call in (lambda g: norm.rms_norm(g(x), w), lambda g: norm.rms_norm(x, g(w)),
                 lambda g: norm.rms_norm(x, w, residual=g(x))[0],
                 lambda g: norm.rms_norm_int8(g(x), g(w), rotate=False)[0], lambda g: moe.route(g(lg), 4)[1],
                 lambda g: moe.route(lg, 4, bias=g(w))[1], lambda g: rope.rotate_axes(g(q), None, p, f)[0],
                 lambda g: rope.rotate_axes(q, None, g(p), f)[0]):
        assert torch.equal(call(neg), call(torch.neg))
    for v, call in ((x, lambda a: norm.rms_norm(a, w)), (lg, lambda a: moe.route(a, 4)[1]),
                    (q, lambda a: rope.rotate_axes(a, None, p, f)[0])):
        a = v.clone().requires_grad_()
        y = call(a)
        d = randn(*y.shape, seed=7).to(dev)
        g1, = torch.autograd.grad(y, a, neg(d), retain_graph=True)
        g2, = torch.autograd.grad(y, a, -d)
        assert torch.equal(g1, g2)


def test_changed_after_the_forward_pass(dev):
    """A tensor that the gradient needs and that is written before it is an error."""
    x, w = randn(4, 64, seed=1).to(dev).requires_grad_(), randn(64, seed=2).to(dev)
    y, h = norm.rms_norm(x, w, residual=x.detach())
    h.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    lg = randn(4, 16, seed=3).to(dev).requires_grad_()
    ids, wt = moe.route(lg, 2)
    assert not ids.requires_grad
    ids.zero_()
    with pytest.raises(RuntimeError, match="inplace"):
        wt.sum().backward()
