"""The bias gradient of the MXFP4 linear, dy's column sums in fp32 rounded once to the
bias's type, against 64 bits, through both host paths and in a captured step."""

import pytest
import torch

from mx_util import DTYPES, assert_close, big_memory, randn  # noqa: F401
from xpu_kernels import mxfp4
from xpu_kernels.int8 import _lib as L

pytestmark = pytest.mark.gpu


def dbias(dev, dy, n, bias_dtype, k=32):
    """The gradient for a dy [M, N], checked to be the same through both host paths."""
    codes, scales = mxfp4.quantize(randn(n, k, seed=3).to(dev))
    x = torch.ones(dy.shape[0], k, dtype=dy.dtype, device=dev)
    b = torch.zeros(n, dtype=bias_dtype, device=dev, requires_grad=True)
    got, = torch.autograd.grad(mxfp4.linear(x, codes, scales, b), b, dy)
    host, L.HOST = L.HOST, None
    try:
        slow, = torch.autograd.grad(mxfp4.linear(x, codes, scales, b), b, dy)
    finally:
        L.HOST = host
    assert got.dtype == bias_dtype and got.shape == (n,)
    assert torch.equal(got.view(torch.uint8), slow.view(torch.uint8))    # (NaNs too)
    return got


@pytest.mark.parametrize("bias_dtype", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n", [(1, 1), (3, 16), (31, 17), (32, 64), (33, 129), (300, 48),
                                 (1025, 2056), (500, 4112)])
def test_bias_gradient(dev, dtype, bias_dtype, m, n):
    """Sums of positive terms, whose fp32 value a 16-bit type does not hold."""
    dy = (randn(m, n, seed=m, dtype=dtype).abs() + 1).to(dev)
    d = dy.cpu().double()
    assert_close(dbias(dev, dy, n, bias_dtype), d.sum(0), d.abs().sum(0), m)


@pytest.mark.parametrize("dtype", DTYPES)
def test_bias_gradient_past_a_16_bit_types_range(dev, dtype):
    """A column sum beyond fp16 is finite in an fp32 or bf16 bias: 300 terms of 300."""
    dy = torch.full((300, 40), 300.0, dtype=dtype, device=dev)
    for bias_dtype in (torch.float32, torch.bfloat16):
        got = dbias(dev, dy, 40, bias_dtype)
        assert torch.equal(got, torch.full_like(got, 90000.0))
    assert dbias(dev, dy, 40, torch.float16).isinf().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_bias_gradient_of_strided_dy(dev, dtype):
    base = randn(50, 96, seed=4, dtype=dtype).to(dev)
    for dy in (base[:, :64], base[:, 3:67], base[:, ::2][:, :40], base[:, :1].expand(50, 64),
               base[:1, :64].expand(50, 64), base[:, :1].expand(50, 9), base[:40, :50].t()):
        d = dy.cpu().double()
        assert_close(dbias(dev, dy, dy.shape[1], torch.float32), d.sum(0), d.abs().sum(0), dy.shape[0])


def test_bias_gradient_specials(dev):
    dy = randn(70, 50, seed=4)
    dy[3, 7], dy[60, 8], dy[5, 9], dy[6, 9] = float("nan"), float("inf"), float("inf"), -float("inf")
    got = dbias(dev, dy.to(dev), 50, torch.float32).cpu()
    assert got.isnan().nonzero().flatten().tolist() == [7, 9] and got[8] == float("inf")


@pytest.mark.parametrize("dtype", DTYPES)
def test_bias_gradient_of_many_rows(dev, big_memory, dtype):
    """More blocks of 32 rows than one dimension of a launch has: sums of ones, exact in fp32."""
    m = 65535 * 32 + 33
    got = dbias(dev, torch.ones(1, 1, dtype=dtype, device=dev).expand(m, 9), 9, torch.float32)
    assert (got == m).all()


def test_bias_gradient_of_no_rows(dev):
    codes, scales = mxfp4.quantize(randn(8, 64).to(dev))
    b = torch.zeros(8, device=dev, requires_grad=True)
    y = mxfp4.linear(torch.empty(0, 64, device=dev), codes, scales, b)
    assert torch.equal(torch.autograd.grad(y.sum(), b)[0], torch.zeros(8, device=dev))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n", [(40, 272), (3000, 72)])
def test_gradients_in_a_graph(dev, dtype, m, n):
    """A captured forward and backward replays with new inputs, eager work in between."""
    k = 288
    codes, scales = mxfp4.quantize(randn(n, k, seed=5).to(dev))
    x = randn(m, k, seed=1, dtype=dtype).to(dev).requires_grad_()
    b = randn(n, seed=2).to(dev).requires_grad_()
    dy = randn(m, n, seed=3, dtype=dtype).to(dev)

    def step():
        y = mxfp4.linear(x, codes, scales, b)
        return (y, *torch.autograd.grad(y, (x, b), dy))

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
        with torch.no_grad():
            x.copy_(randn(m, k, seed=seed, dtype=dtype))
        dy.copy_(randn(m, n, seed=seed + 9, dtype=dtype))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in out]
        for g, w in zip(got, step()):
            assert torch.equal(g, w)
