"""int8.linear_quantized: what its inputs are beside their values."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from mx_util import randn
from xpu_kernels import int8

pytestmark = pytest.mark.gpu


def inputs(dev):
    q, s = int8.quantize(randn(5, 256, seed=1).bfloat16().to(dev))
    w8, ws = int8.prepare_weight(randn(32, 256, seed=2).bfloat16().to(dev), pack=False)
    return [q, s, w8, ws, randn(32, seed=3).to(dev)]


@pytest.mark.parametrize("which", range(5))
def test_lazily_negated(dev, which):
    args, negated = inputs(dev), inputs(dev)
    args[which] = torch.neg(args[which])
    negated[which] = torch._neg_view(negated[which])
    assert torch.equal(int8.linear_quantized(*negated), int8.linear_quantized(*args))


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("packed", [False, True])
def test_lazily_negated_beside_it(dev, which, packed):
    """The int8 calls that share its arguments."""
    x, args = randn(5, 256, seed=1).bfloat16().to(dev), inputs(dev)[2:]
    args = [x, *args]
    if packed:
        int8.pack_weight(args[1])
    negated = list(args)
    args[which] = torch.neg(args[which])
    negated[which] = torch._neg_view(negated[which])
    assert torch.equal(int8.linear(*negated), int8.linear(*args))
    assert torch.equal(int8.int_mm(inputs(dev)[0], negated[1].t()), int8.int_mm(inputs(dev)[0], args[1].t()))
    acc = int8.int_mm(inputs(dev)[0], args[1].t())
    assert torch.equal(int8.dequant_slice(torch._neg_view(acc), *inputs(dev)[1:4:2]),
                       int8.dequant_slice(-acc, *inputs(dev)[1:4:2]))
    if which == 0:
        for a, b in zip(int8.quantize(negated[0]), int8.quantize(args[0])):
            assert torch.equal(a, b)
        for a, b in zip(int8.prepare_weight(negated[0][:, None].expand(5, 16, 256).reshape(80, 256)),
                        int8.prepare_weight(args[0][:, None].expand(5, 16, 256).reshape(80, 256))):
            assert torch.equal(a, b)


@pytest.mark.parametrize("which", [1, 3, 4])
def test_tangents(dev, which):
    args = inputs(dev)
    with fwad.dual_level():
        args[which] = fwad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            int8.linear_quantized(*args)
