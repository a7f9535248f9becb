"""Forward-mode derivatives: the operators have none, and say so."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from mx_util import DTYPES, randn, router
from xpu_kernels import moe, mxfp4
from xpu_kernels.int8 import _lib as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("dtype", DTYPES)
def test_forward_mode_is_refused(dev, monkeypatch, dtype, grad, native):
    t, top, e, k, n = 6, 2, 4, 64, 48
    w, s = mxfp4.quantize(randn(n, k, seed=1).to(dev))
    ws, ss = mxfp4.quantize(randn(e, n, k, seed=2).to(dev))
    up, down = mxfp4.quantize(randn(e, 2 * k, k, seed=6).to(dev)), mxfp4.quantize(randn(e, k, k, seed=7).to(dev))
    ids = router(t, top, e, seed=3).to(dev)
    routing = moe.sort(ids, e)
    x, z = randn(t, k, seed=4, dtype=dtype).to(dev), randn(t * top, k, seed=5, dtype=dtype).to(dev)
    b, weights = torch.zeros(n, device=dev), torch.rand(t, top, device=dev)
    if not native:
        monkeypatch.setattr(L, "HOST", None)
    calls = {
        "linear x": (x, lambda v: mxfp4.linear(v, w, s, b)),
        "linear bias": (b, lambda v: mxfp4.linear(x, w, s, v)),
        "experts": (z, lambda v: mxfp4.grouped_linear(v, ws, ss, routing)),
        "experts, gathering": (x, lambda v: mxfp4.grouped_linear(v, ws, ss, routing, gather=True)),
        "dispatch": (x, lambda v: moe.dispatch(v, routing)),
        "combine z": (z, lambda v: moe.combine(v, routing, weights)),
        "combine weights": (weights, lambda v: moe.combine(z, routing, v)),
        "combine 16-bit weights": (weights.bfloat16(), lambda v: moe.combine(z, routing, v)),
        "ffn x": (x, lambda v: moe.ffn(v, ids, weights, up, down)),
        "ffn weights": (weights, lambda v: moe.ffn(x, ids, v, up, down)),
    }
    for name, (v, call) in calls.items():
        with fwad.dual_level(), torch.set_grad_enabled(grad):
            call(v)                                        # an open level alone changes nothing
            with pytest.raises(NotImplementedError, match="forward-mode"):
                print(name, call(fwad.make_dual(v, torch.ones_like(v))))
        call(v)


def test_quantization_has_no_derivative(dev):
    """Codes and scales are whole numbers: the tangent ends there, as a gradient does."""
    x = randn(4, 64, seed=1).to(dev)
    with fwad.dual_level():
        codes, scales = mxfp4.quantize(fwad.make_dual(x, torch.ones_like(x)))
    want = mxfp4.quantize(x)
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])


def test_function_transforms_are_refused(dev):
    w, s = mxfp4.quantize(randn(48, 64, seed=1).to(dev))
    x = randn(4, 64, seed=2).to(dev)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda v: mxfp4.linear(v, w, s), (x,), (x,))
