"""The memory that a gradient takes beside its result: none for a dy that the kernels read
where it lies."""

import pytest
import torch

from mx_util import randn, router
from xpu_kernels import moe, mxfp4
from xpu_kernels.int8 import _lib as L

pytestmark = pytest.mark.gpu


def peak(fn):
    """The most bytes that fn held beyond what was there before it."""
    fn()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    fn()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("native", [True, False])
def test_experts_gradient_keeps_no_copy_of_dy(dev, monkeypatch, native):
    t, top, e, k, n = 512, 2, 8, 256, 4096
    codes, scales = mxfp4.quantize(randn(e, n, k, seed=5).to(dev))
    routing = moe.sort(router(t, top, e, seed=3).to(dev), e)
    x = randn(t * top, k, seed=1, dtype=torch.bfloat16).to(dev).requires_grad_()
    y = mxfp4.grouped_linear(x, codes, scales, routing)
    dy = randn(t * top, n, seed=2, dtype=torch.bfloat16).to(dev)      # 8 MiB, dx 0.5
    if not native:
        monkeypatch.setattr(L, "HOST", None)
        y = mxfp4.grouped_linear(x, codes, scales, routing)
    held = peak(lambda: torch.autograd.grad(y, x, dy, retain_graph=True))
    assert held < dy.numel(), f"{held} bytes beside a dy of {2 * dy.numel()}"


@pytest.mark.parametrize("native", [True, False])
def test_linear_gradient_keeps_no_copy_of_dy(dev, monkeypatch, native):
    """One weight, at a shape whose dx is taken from the 4-bit weight in tiles."""
    m, k, n = 64, 8192, 2048
    codes, scales = mxfp4.quantize(randn(n, k, seed=5).to(dev))
    if not native:
        monkeypatch.setattr(L, "HOST", None)
    x = randn(m, k, seed=1, dtype=torch.bfloat16).to(dev).requires_grad_()
    y = mxfp4.linear(x, codes, scales)
    dy = randn(m, n, seed=2, dtype=torch.bfloat16).to(dev)            # 256 KiB, dx 1 MiB
    held = peak(lambda: torch.autograd.grad(y, x, dy, retain_graph=True))
    assert held < 2 * m * k + dy.numel(), f"{held} bytes with a dx of {2 * m * k}"
