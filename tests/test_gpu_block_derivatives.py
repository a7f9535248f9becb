"""The inputs beside the heads, rows and logits of the operators between a block's projections:
derivatives that these do not have are refused, not left out, and signs are applied."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from mx_util import randn
from xpu_kernels import int8, rope
from xpu_kernels.int8 import _lib as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("both", [True, False])
def test_frequencies_and_positions(dev, monkeypatch, native, both):
    if not native:
        monkeypatch.setattr(L, "HOST", None)
    q = randn(1, 3, 2, 16, seed=4).to(dev).requires_grad_(both)
    f, p = rope.axis_frequencies((8,), device=dev), torch.rand(1, 3, device=dev)
    learnt = rope.AxisFrequencies(f.inv_freq.clone().requires_grad_(), f.axis)
    with pytest.raises(ValueError, match="no gradient"):
        rope.rotate_axes(q, None, p, learnt)
    with torch.no_grad():
        turned = rope.rotate_axes(q, None, p, learnt)[0]
    assert torch.equal(turned, rope.rotate_axes(q, None, p, f)[0])
    with fwad.dual_level():
        for pos, freq in ((fwad.make_dual(p, torch.ones_like(p)), f),
                          (p, rope.AxisFrequencies(fwad.make_dual(f.inv_freq, torch.ones_like(f.inv_freq)), f.axis))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                rope.rotate_axes(q, None, pos, freq)


@pytest.mark.parametrize("native", [True, False])
def test_lazily_negated_frequencies(dev, monkeypatch, native):
    """A sign that is a flag of the view is applied."""
    if not native:
        monkeypatch.setattr(L, "HOST", None)
    q, p = randn(1, 3, 2, 16, seed=4).to(dev), torch.arange(3, device=dev)[None]
    f = rope.axis_frequencies((4, 4), device=dev)
    for i in range(2):
        view = [torch._neg_view(t) if i == j else t for j, t in enumerate(f)]
        made = [-t if i == j else t for j, t in enumerate(f)]
        assert torch.equal(rope.rotate_axes(q, None, p, rope.AxisFrequencies(*view))[0],
                           rope.rotate_axes(q, None, p, rope.AxisFrequencies(*made))[0])
