"""Products and gradients with scales at the ends of their range."""

import pytest
import torch

import oracle.mxfp4 as O
from mx_util import assert_close, randn
from xpu_kernels import mxfp4

pytestmark = pytest.mark.gpu


def weight(dev, n, k, exponents, seed=3):
    """Random codes with the scale bytes of ``exponents``, a value a row by turns."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scales = torch.full((n, O.scale_width(k)), 127, dtype=torch.uint8)
    scales[:, :k // 32] = torch.tensor(exponents, dtype=torch.uint8).repeat(-(-n // len(exponents)))[:n, None]
    return codes.to(dev), scales.to(dev), O.dequantize(codes, scales)


@pytest.mark.parametrize("m", [1, 12, 40, 200, 2000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_products_of_the_smallest_and_largest_scales(dev, dtype, m):
    """2^-127 and 2^-126 on one side (bf16's subnormals) with large ones on the other."""
    k, n = 288, 264
    codes, scales, wq = weight(dev, n, k, [0, 1, 2, 127, 150])
    x = randn(m, k, seed=m).to(dtype)
    x[0::3] *= 2.0 ** 80                                   # (no sum past fp32's range)
    x[1::3] *= 2.0 ** -100
    y = mxfp4.linear(x.to(dev), codes, scales)
    xq = O.dequantize(*O.quantize(x))
    assert_close(y, xq @ wq.t(), xq.abs() @ wq.abs().t(), k)
    codes, scales, wq = weight(dev, n, k, [254, 253, 240])
    x = (randn(m, k, seed=m) * 2.0 ** -120).to(dtype)
    x[0::2] *= 2.0 ** -9                                   # subnormal, scale 2^-127
    y = mxfp4.linear(x.to(dev), codes, scales)
    xq = O.dequantize(*O.quantize(x))
    assert_close(y, xq @ wq.t(), xq.abs() @ wq.abs().t(), k)


@pytest.mark.parametrize("m,n", [(8, 264), (300, 264), (300, 2064), (2000, 4096)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_of_the_smallest_and_largest_scales(dev, dtype, m, n):
    k = 288
    codes, scales, wq = weight(dev, n, k, [0])
    x = randn(m, k, seed=1).to(dtype).to(dev).requires_grad_()
    dy = (randn(m, n, seed=m) * 2.0 ** 110).to(dtype)
    dx, = torch.autograd.grad(mxfp4.linear(x, codes, scales), x, dy.to(dev))
    d = dy.double()
    assert_close(dx, d @ wq, d.abs() @ wq.abs(), 3 * n)
    codes, scales, wq = weight(dev, n, k, [230])
    dy = (randn(m, n, seed=m) * 2.0 ** -128).to(dtype)     # subnormal
    dx, = torch.autograd.grad(mxfp4.linear(x, codes, scales), x, dy.to(dev))
    # of an fp32's bits those below bf16's least subnormal, 2^-133, are dropped
    d = torch.trunc(dy.double() * 2.0 ** 133) * 2.0 ** -133
    assert_close(dx, d @ wq, d.abs() @ wq.abs(), 3 * n)
