"""MXFP4 on the device against the 64-bit oracle: quantization bit for bit, the
products and gradients within the bound of fp32 sums and one rounding."""

import pytest
import torch

import oracle.mxfp4 as O
from mx_util import DTYPES, assert_close, big_memory, randn, router  # noqa: F401
from xpu_kernels import moe, mxfp4

pytestmark = pytest.mark.gpu


def same_bits(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.uint8), b.cpu().contiguous().view(torch.uint8))


# ------------------------------------------------------------------ quantize
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 32), (1, 4096), (3, 480), (17, 512), (5, 544), (130, 1280),
                                 (257, 96), (2048, 4128)])
def test_quantize_bit_for_bit(dev, dtype, m, k):
    x = randn(m, k, seed=m + k, dtype=dtype)
    x[:, ::37] *= 30
    codes, scales = mxfp4.quantize(x.to(dev))
    oc, os_ = O.quantize(x)
    assert torch.equal(codes.cpu(), oc) and torch.equal(scales.cpu(), os_)
    for out in DTYPES:
        v = mxfp4.dequantize(codes, scales, out)
        assert v.dtype == out and same_bits(v, O.dequantize(oc, os_).to(out))


def test_quantize_every_bf16(dev):
    """Each finite bf16 as a block's maximum and beside one of every binade above it."""
    b = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    b = b[torch.isfinite(b)]
    x = torch.zeros(b.numel(), 32, dtype=torch.bfloat16)
    x[:, 0] = b
    for i in range(1, 8):
        x[:, i] = (b.double() * 2.0 ** -i).to(torch.bfloat16)
    x[:, 8:] = b[:, None] * torch.rand(24, generator=torch.Generator().manual_seed(3))
    codes, scales = mxfp4.quantize(x.to(dev))
    oc, os_ = O.quantize(x)
    assert torch.equal(scales.cpu(), os_) and torch.equal(codes.cpu(), oc)


def test_quantize_ties_fp32(dev):
    """fp32 values on, one ulp below and one above every rounding boundary."""
    mids = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5., 6., 7., 7.999])
    below = torch.nextafter(mids, torch.zeros(()))
    above = torch.nextafter(mids, torch.full((), 9.0))
    row = torch.cat([mids, below, above, torch.tensor([4.0, -0.0])])
    x = torch.stack([row * s * 2.0 ** e for s in (1, -1) for e in (-130, -126, -20, 0, 40, 124)])
    codes, scales = mxfp4.quantize(x.to(dev))
    oc, os_ = O.quantize(x)
    assert torch.equal(codes.cpu(), oc) and torch.equal(scales.cpu(), os_)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_specials(dev, dtype):
    x = torch.ones(6, 96, dtype=dtype)
    x[0, 40] = float("inf")
    x[1, 0] = float("nan")
    x[2, 95] = -float("inf")
    x[3] = 0
    x[4, 32:64] = torch.finfo(dtype).max
    x[5] = torch.finfo(dtype).tiny / 4
    codes, scales = mxfp4.quantize(x.to(dev))
    _, os_ = O.quantize(x)
    assert torch.equal(scales.cpu(), os_)
    v = mxfp4.dequantize(codes, scales, torch.float32).cpu()
    for row, block in ((0, 1), (1, 0), (2, 2)):
        nan = v[row].isnan().reshape(3, 32).all(-1)
        assert nan.tolist() == [i == block for i in range(3)]
    assert (v[3] == 0).all() and torch.isfinite(v[3:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_strides(dev, dtype):
    base = randn(40, 300, seed=4, dtype=dtype).to(dev)
    for x in (base[:, :288], base[:, 5:293], base[1::3, 4:68], base[:, :40].t()[:, :32],
              base[:32, :64].expand(2, 32, 64), base[:, ::2][:, :128], base[3, 1:65]):
        codes, scales = mxfp4.quantize(x)
        oc, os_ = O.quantize(x)
        assert torch.equal(codes.cpu(), oc) and torch.equal(scales.cpu(), os_)


def test_quantize_empty(dev):
    codes, scales = mxfp4.quantize(torch.empty(0, 64, device=dev))
    assert codes.shape == (0, 32) and scales.shape == (0, 16)
    assert mxfp4.dequantize(codes, scales).shape == (0, 64)


def test_quantize_past_4_gib(dev, big_memory):
    m, k = 70001, 32768                                   # 4.6 GB of bf16
    x = torch.empty(m, k, dtype=torch.bfloat16, device=dev).normal_(generator=torch.Generator(dev).manual_seed(1))
    codes, scales = mxfp4.quantize(x)
    v = mxfp4.dequantize(codes, scales)
    for r in (slice(0, 3), slice(65534, 65539), slice(m - 3, m)):
        oc, os_ = O.quantize(x[r])
        assert torch.equal(codes[r].cpu(), oc) and torch.equal(scales[r].cpu(), os_)
        assert same_bits(v[r], O.dequantize(oc, os_).to(torch.bfloat16))


def test_pad_scales(dev):
    x = randn(6, 96, seed=8).to(dev)
    codes, scales = mxfp4.quantize(x)
    assert torch.equal(mxfp4.pad_scales(scales[:, :3]), scales)


# -------------------------------------------------------------------- linear
def weight(n, k, seed, dev):
    w = randn(n, k, seed=seed, scale=0.05)
    return mxfp4.quantize(w.to(dev)), O.dequantize(*O.quantize(w))


def check_linear(dev, x, n, bias=None, seed=1, alter=None):
    k = x.shape[-1]
    (codes, scales), wq = weight(n, k, seed, dev)
    if alter:
        alter(scales)
    xq = O.dequantize(*O.quantize(x))
    y = mxfp4.linear(x.to(dev) if not x.is_cuda else x, codes, scales,
                     None if bias is None else bias.to(dev))
    assert y.dtype == x.dtype and y.shape == (*x.shape[:-1], n)
    want, mag = xq @ wq.t(), xq.abs() @ wq.abs().t()
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    assert_close(y, want, mag, k + 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(1, 32, 1), (1, 4096, 256), (3, 544, 17), (16, 1024, 48),
                                   (17, 1024, 48), (33, 4640, 130), (100, 288, 264),
                                   (129, 1280, 127), (300, 800, 513), (257, 2048, 1000)])
def test_linear(dev, dtype, m, k, n):
    x = randn(m, k, seed=m, dtype=dtype)
    x[:, 3::41] *= 20
    check_linear(dev, x, n, bias=randn(n, seed=2, dtype=dtype))


@pytest.mark.parametrize("dtype,m,k,n", [
    (torch.bfloat16, 1, 2048, 8209), (torch.float16, 16, 4096, 8232), (torch.float32, 2, 8192, 8200),
    (torch.bfloat16, 9, 8224, 40), (torch.float32, 5, 16416, 72), (torch.float16, 3, 4128, 16500),
    (torch.float16, 32, 2080, 4111), (torch.bfloat16, 33, 2048, 8212), (torch.float32, 17, 8256, 56),
    (torch.bfloat16, 64, 4128, 4200), (torch.float16, 49, 12320, 4112), (torch.float32, 65, 640, 200)])
def test_linear_few_rows(dev, dtype, m, k, n):
    """One to four blocks of 16 rows, K on both sides of what a block's waves hold, weights
    with several and ragged blocks of rows each."""
    x = randn(m, k, seed=m, dtype=dtype)
    x[:, 5::37] *= 30
    check_linear(dev, x, n, bias=randn(n, seed=2, dtype=dtype))


@pytest.mark.parametrize("dtype,m,k,n", [
    (torch.bfloat16, 130, 4096, 520), (torch.float16, 300, 3104, 1040), (torch.float32, 500, 2048, 264),
    (torch.bfloat16, 97, 8192, 1000), (torch.bfloat16, 33, 16416, 40), (torch.float16, 64, 8224, 4120),
    (torch.bfloat16, 511, 4128, 72)])
def test_linear_several_blocks_of_few_rows(dev, dtype, m, k, n):
    """More rows than a block of the kernel of few rows takes, K on both sides of what its
    waves hold."""
    x = randn(m, k, seed=m, dtype=dtype)
    check_linear(dev, x, n, bias=randn(n, seed=2, dtype=dtype))


@pytest.mark.parametrize("t,top,experts,k,n,dropped", [
    (3, 3, 40, 2080, 2056, 0.0), (60, 4, 10, 544, 300, 0.1), (60, 4, 10, 4160, 136, 0.1),
    (100, 5, 9, 288, 520, 0.05), (70, 6, 8, 4128, 72, 0.0), (31, 2, 4, 8224, 40, 0.2)])
def test_grouped_few_rows(dev, t, top, experts, k, n, dropped):
    """Groups of fewer and of more rows than a block takes."""
    ids = router(t, top, experts, seed=t, dropped=dropped)
    routing = moe.sort(ids.to(dev), experts)
    _, _, orows, ooff = O.sort(ids, experts)
    codes, scales = mxfp4.quantize(randn(experts, n, k, seed=7, scale=0.05).to(dev))
    wq = O.dequantize(codes.cpu(), scales.cpu())
    for gather in (False, True):
        x = randn(t if gather else t * top, k, seed=8, dtype=torch.bfloat16)
        rows = orows if gather else torch.arange(t * top, dtype=torch.int32)
        xq = O.dequantize(*O.quantize(x))
        y = mxfp4.grouped_linear(x.to(dev), codes, scales, routing, gather=gather)
        assert_close(y, O.grouped(xq, wq, rows, ooff), O.grouped(xq.abs(), wq.abs(), rows, ooff), k)


@pytest.mark.parametrize("dtype,m,k,n", [(torch.bfloat16, 4090, 8160, 4080),
                                         (torch.bfloat16, 4001, 8192, 4081),
                                         (torch.float32, 3890, 7968, 4096)])
def test_linear_large_tiles(dev, big_memory, dtype, m, k, n):
    """Shapes that take the large tiles, ragged in every dimension."""
    x = randn(m, k, seed=m, dtype=dtype)
    bias = randn(n, seed=2, dtype=dtype)
    (codes, scales), wq = weight(n, k, 1, dev)
    xq, wd = O.dequantize(*O.quantize(x)).to(dev), wq.to(dev)
    y = mxfp4.linear(x.to(dev), codes, scales, bias.to(dev))
    b = bias.to(dev).double()
    assert_close(y, (xq @ wd.t() + b).cpu(), (xq.abs() @ wd.abs().t() + b.abs()).cpu(), k + 1)


@pytest.mark.parametrize("gather", [False, True])
def test_grouped_large_tiles(dev, big_memory, gather):
    t, top, e, k, n = 4095, 2, 3, 8160, 3800
    ids = router(t, top, e, seed=1, dropped=0.02)
    routing = moe.sort(ids.to(dev), e)
    w = randn(e, n, k, seed=7, scale=0.05)
    codes, scales = mxfp4.quantize(w.to(dev))
    x = randn(t if gather else t * top, k, seed=8, dtype=torch.bfloat16)
    y = mxfp4.grouped_linear(x.to(dev), codes, scales, routing, gather=gather)
    xq = O.dequantize(*O.quantize(x)).to(dev)
    off = routing.offsets.tolist()
    for i in range(e):
        r = slice(off[i], off[i + 1])
        xr = xq[routing.rows[r].long()] if gather else xq[r]
        wq = O.dequantize(codes[i], scales[i]).to(dev)
        assert_close(y[r], (xr @ wq.t()).cpu(), (xr.abs() @ wq.abs().t()).cpu(), k)
    assert (y[off[-1]:] == 0).all()


@pytest.mark.parametrize("m", [1, 40, 200])
@pytest.mark.parametrize("bias_dtype", DTYPES)
def test_linear_bias_types(dev, m, bias_dtype):
    check_linear(dev, randn(m, 160, seed=m, dtype=torch.bfloat16), 50,
                 bias=randn(50, seed=2, dtype=bias_dtype))


@pytest.mark.parametrize("m", [2, 20, 150])
def test_linear_padding_scales_are_unused(dev, m):
    """The bytes past K/32 may hold anything, the NaN byte among them."""
    def alter(scales):
        scales[:, 800 // 32:] = 255
    check_linear(dev, randn(m, 800, seed=m), 40, alter=alter)


@pytest.mark.parametrize("m", [1, 5, 70, 300])
def test_linear_specials(dev, m):
    """A NaN block of x is NaN in its row alone, one of the weight in its column;
    values at the top of the range overflow to infinities as sums do."""
    k, n = 1056, 70
    x = randn(m, k, seed=5)
    (codes, scales), wq = weight(n, k, 6, dev)
    x[m // 2, 700] = float("inf")
    scales[7, 32] = 255
    y = mxfp4.linear(x.to(dev), codes, scales).cpu()
    nan = torch.zeros(m, n, dtype=torch.bool)
    nan[m // 2] = True
    nan[:, 7] = True
    assert torch.equal(y.isnan(), nan)
    x = torch.full((m, k), 3e38)
    (codes, scales), wq = weight(n, k, 6, dev)
    y = mxfp4.linear(x.to(dev), codes, scales).cpu()
    assert (y.isinf() | (y.abs() > 1e37)).float().mean() > 0.9


@pytest.mark.parametrize("m", [2, 30, 200])
def test_linear_strides_and_shapes(dev, m):
    base = randn(m + 3, 700, seed=9, dtype=torch.bfloat16).to(dev)
    for x in (base[:m, :640], base[3:, 3:643], base[:m, 1:513]):
        check_linear(dev, x, 96)
    check_linear(dev, base[:m, :640].reshape(1, m, 640).expand(3, m, 640), 33)
    w, s = mxfp4.quantize(randn(96, 640, seed=1, scale=0.05).to(dev))
    wide = torch.zeros(96, 400, dtype=torch.uint8, device=dev)
    wide[:, 3:323] = w
    assert torch.equal(mxfp4.linear(base[:m, :640], wide[:, 3:323], s),
                       mxfp4.linear(base[:m, :640], w, s))


def test_linear_empty(dev):
    codes, scales = mxfp4.quantize(randn(8, 64).to(dev))
    assert mxfp4.linear(torch.empty(0, 64, device=dev), codes, scales).shape == (0, 8)
    x = torch.empty(2, 0, 64, device=dev, requires_grad=True)
    y = mxfp4.linear(x, codes, scales)
    y.sum().backward()
    assert x.grad.shape == x.shape


def test_linear_on_another_stream(dev):
    x = randn(200, 512, seed=3, dtype=torch.bfloat16).to(dev)
    codes, scales = mxfp4.quantize(randn(300, 512, seed=4).to(dev))
    want = mxfp4.linear(x, codes, scales)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = mxfp4.linear(x, codes, scales)
    s.synchronize()
    assert torch.equal(y, want)


# ----------------------------------------------------------------- gradients
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(1, 32, 1), (7, 96, 40), (130, 544, 72), (200, 288, 129),
                                   (65, 1280, 512), (300, 160, 333)])
def test_linear_gradients(dev, dtype, m, k, n):
    x = randn(m, k, seed=m, dtype=dtype).to(dev).requires_grad_()
    bias = randn(n, seed=2, dtype=dtype).to(dev).requires_grad_()
    (codes, scales), wq = weight(n, k, 3, dev)
    dy = randn(m, n, seed=4, dtype=dtype)
    y = mxfp4.linear(x, codes, scales, bias)
    dx, db = torch.autograd.grad(y, (x, bias), dy.to(dev))
    d = dy.double()
    assert dx.dtype == dtype and db.dtype == dtype
    assert_close(dx, d @ wq, d.abs() @ wq.abs(), 3 * n)
    assert_close(db, d.sum(0), d.abs().sum(0), m + 1)


@pytest.mark.parametrize("m,k,n", [(127, 96, 64), (128, 96, 64), (129, 1056, 272), (128, 96, 72),
                                   (700, 2080, 1040)])
def test_linear_gradient_of_many_rows(dev, m, k, n):
    """Gradients of a bf16 product of more rows than a tile, contiguous and strided."""
    (codes, scales), wq = weight(n, k, 3, dev)
    x = randn(m, k, seed=m, dtype=torch.bfloat16).to(dev).requires_grad_()
    y = mxfp4.linear(x, codes, scales)
    base = randn(m, n + 24, seed=4, dtype=torch.bfloat16).to(dev)
    for dy in (base[:, :n].contiguous(), base[:, :n], base[:, 3:n + 3], base[:, :1].expand(m, n)):
        dx, = torch.autograd.grad(y, x, dy, retain_graph=True)
        d = dy.cpu().double()
        assert_close(dx, d @ wq, d.abs() @ wq.abs(), 3 * n)


@pytest.mark.parametrize("m,k,n", [(1, 512, 1536), (1, 512, 1472), (5, 96, 4096), (16, 512, 2560),
                                   (300, 512, 4096), (65, 2080, 4112), (129, 544, 4104)])
def test_linear_gradient_of_long_contractions(dev, m, k, n):
    """Both sides of the sizes at which dx of a bf16 product is taken from the weight read
    back, contiguous and strided."""
    (codes, scales), wq = weight(n, k, 3, dev)
    x = randn(m, k, seed=m, dtype=torch.bfloat16).to(dev).requires_grad_()
    y = mxfp4.linear(x, codes, scales)
    base = randn(m, n + 24, seed=4, dtype=torch.bfloat16).to(dev)
    for dy in (base[:, :n].contiguous(), base[:, :n], base[:, 3:n + 3], base[:, :1].expand(m, n)):
        dx, = torch.autograd.grad(y, x, dy, retain_graph=True)
        d = dy.cpu().double()
        assert_close(dx, d @ wq, d.abs() @ wq.abs(), 3 * n)


@pytest.mark.parametrize("dtype,m,k,n", [
    (torch.float16, 64, 4224, 136), (torch.float16, 65, 33056, 72), (torch.float32, 31, 160, 200),
    (torch.float32, 33, 1056, 1000), (torch.bfloat16, 64, 96, 1032), (torch.float16, 260, 16416, 40)])
def test_linear_gradient_in_tiles_of_few_rows(dev, dtype, m, k, n):
    """Row and column ends of the small tiles, one piece of dy and several, and shapes
    that go to the larger ones."""
    (codes, scales), wq = weight(n, k, 3, dev)
    x = randn(m, k, seed=m, dtype=dtype).to(dev).requires_grad_()
    dy = randn(m, n, seed=4, dtype=dtype)
    dx, = torch.autograd.grad(mxfp4.linear(x, codes, scales), x, dy.to(dev))
    d = dy.double()
    assert_close(dx, d @ wq, d.abs() @ wq.abs(), 3 * n)


@pytest.mark.parametrize("t,top,experts,k,n,dropped", [
    (50, 2, 3, 1056, 264, 0.1), (97, 2, 3, 160, 520, 0.0), (700, 1, 11, 288, 72, 0.1), (33, 1, 1, 96, 1000, 0.0)])
def test_grouped_gradient_of_few_rows(dev, t, top, experts, k, n, dropped):
    """Groups on both sides of 32 and 64 rows."""
    ids = router(t, top, experts, seed=t, dropped=dropped)
    routing = moe.sort(ids.to(dev), experts)
    _, opos, orows, ooff = O.sort(ids, experts)
    codes, scales = mxfp4.quantize(randn(experts, n, k, seed=7, scale=0.05).to(dev))
    wt = O.dequantize(codes.cpu(), scales.cpu()).transpose(1, 2)
    r = t * top
    x = randn(r, k, seed=8, dtype=torch.bfloat16).to(dev).requires_grad_()
    dy = randn(r, n, seed=9, dtype=torch.bfloat16)
    dx, = torch.autograd.grad(mxfp4.grouped_linear(x, codes, scales, routing), x, dy.to(dev))
    d, same = dy.double(), torch.arange(r, dtype=torch.int32)
    assert_close(dx, O.grouped(d, wt, same, ooff), O.grouped(d.abs(), wt.abs(), same, ooff), n)


def test_linear_gradient_of_strided_dy(dev):
    x = randn(50, 96, seed=1, dtype=torch.bfloat16).to(dev).requires_grad_()
    (codes, scales), wq = weight(64, 96, 3, dev)
    y = mxfp4.linear(x, codes, scales)
    dy = randn(50, 80, seed=4, dtype=torch.bfloat16).to(dev)
    for d in (dy[:, :64], dy[:, 3:67], dy[:, :1].expand(50, 64), dy[:1, :64].expand(50, 64)):
        dx, = torch.autograd.grad(y, x, d, retain_graph=True)
        want = d.cpu().double()
        assert_close(dx, want @ wq, want.abs() @ wq.abs(), 64)


def test_linear_gradient_against_differences(dev):
    """Where x lies on its grid and its blocks' maxima stay, the product is linear in
    x, and the difference quotient of steps along the grid is the gradient."""
    k, n = 96, 24
    x = torch.ones(k)
    x[::32] = 6.0                                          # scale 1: the grid itself
    codes, scales = mxfp4.quantize(randn(n, k, seed=5).to(dev))
    at = [1, 17, 31, 33, 95]
    plus, minus = x.repeat(len(at), 1), x.repeat(len(at), 1)
    for i, c in enumerate(at):
        plus[i, c] = 1.5
        minus[i, c] = 0.5
    xs = x[None].to(dev).requires_grad_()
    dy = randn(1, n, seed=6).to(dev)
    dx, = torch.autograd.grad(mxfp4.linear(xs, codes, scales), xs, dy)
    rise = ((mxfp4.linear(plus.to(dev), codes, scales) - mxfp4.linear(minus.to(dev), codes, scales))
            .double() @ dy[0].double())
    # fp32 products of a few hundred: K sums of 2^-24 each in either
    assert torch.allclose(rise.cpu(), dx[0, at].double().cpu(), rtol=0,
                          atol=2 * k * 2.0 ** -23 * 6 * 4 * n)


def test_linear_gradient_specials(dev):
    m, n, k = 40, 64, 96
    x = randn(m, k, seed=1).to(dev).requires_grad_()
    codes, scales = mxfp4.quantize(randn(n, k, seed=2).to(dev))
    dy = randn(m, n, seed=3)
    dy[5, 6] = float("nan")
    dy[7, 8] = float("inf")
    dy[9] = torch.finfo(torch.float32).max
    dx, = torch.autograd.grad(mxfp4.linear(x, codes, scales), x, dy.to(dev))
    bad = ~torch.isfinite(dx).all(-1)
    assert bad[5] and bad[7] and not bad[:5].any() and not bad[10:].any()
    assert dx[5].isnan().all()


# ------------------------------------------------------------ experts' products
GROUPED = [
    # t, top, experts, k, n, dropped
    (1, 1, 1, 32, 1, 0.0), (1, 2, 8, 544, 40, 0.0), (4, 4, 32, 1024, 64, 0.0),
    (5, 3, 4, 96, 17, 0.5), (40, 2, 3, 288, 136, 0.1), (200, 4, 8, 800, 130, 0.05),
    (300, 2, 70, 512, 96, 0.2), (64, 1, 1024, 64, 16, 0.1), (150, 8, 2, 160, 264, 0.3),
    (9, 2, 4, 64, 24, 1.0),
]


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("t,top,experts,k,n,dropped", GROUPED)
def test_grouped_linear_and_gradient(dev, t, top, experts, k, n, dropped, gather):
    ids = router(t, top, experts, seed=t, dropped=dropped)
    routing = moe.sort(ids.to(dev), experts)
    _, opos, orows, ooff = O.sort(ids, experts)
    r = t * top
    w = randn(experts, n, k, seed=7, scale=0.05)
    codes, scales = mxfp4.quantize(w.to(dev))
    wq = O.dequantize(*O.quantize(w))
    x = randn(t if gather else r, k, seed=8, dtype=torch.bfloat16)
    rows = orows if gather else torch.arange(r, dtype=torch.int32)
    if not gather and dropped:
        x[int(ooff[-1]):] = float("nan")                   # rows of no expert hold anything
    xq = O.dequantize(*O.quantize(x))
    xd = x.to(dev).requires_grad_()
    y = mxfp4.grouped_linear(xd, codes, scales, routing, gather=gather)
    assert_close(y, O.grouped(xq, wq, rows, ooff), O.grouped(xq.abs(), wq.abs(), rows, ooff), k)
    dy = randn(r, n, seed=9, dtype=torch.bfloat16)
    dx, = torch.autograd.grad(y, xd, dy.to(dev))
    d = dy.double()
    wt = wq.transpose(1, 2)
    dxs = O.grouped(d, wt, torch.arange(r, dtype=torch.int32), ooff)
    mag = O.grouped(d.abs(), wt.abs(), torch.arange(r, dtype=torch.int32), ooff)
    if gather:
        dxs, mag = dxs[opos.long()].sum(1), mag[opos.long()].sum(1)
    assert_close(dx, dxs, mag, n + top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t", [3, 90])
def test_grouped_types(dev, dtype, t):
    test_types = router(t, 2, 4, seed=t)
    routing = moe.sort(test_types.to(dev), 4)
    _, opos, orows, ooff = O.sort(test_types, 4)
    w = randn(4, 50, 96, seed=7, scale=0.05)
    codes, scales = mxfp4.quantize(w.to(dev))
    wq = O.dequantize(*O.quantize(w))
    x = randn(t, 96, seed=8, dtype=dtype)
    xq = O.dequantize(*O.quantize(x))
    xd = x.to(dev).requires_grad_()
    y = mxfp4.grouped_linear(xd, codes, scales, routing, gather=True)
    assert y.dtype == dtype
    assert_close(y, O.grouped(xq, wq, orows, ooff), O.grouped(xq.abs(), wq.abs(), orows, ooff), 96)
    dy = randn(2 * t, 50, seed=9, dtype=dtype)
    dx, = torch.autograd.grad(y, xd, dy.to(dev))
    every = torch.arange(2 * t, dtype=torch.int32)
    dxs = O.grouped(dy.double(), wq.transpose(1, 2), every, ooff)[opos.long()].sum(1)
    mag = O.grouped(dy.double().abs(), wq.transpose(1, 2).abs(), every, ooff)[opos.long()].sum(1)
    assert dx.dtype == dtype
    assert_close(dx, dxs, mag, 3 * 50 + 2)


def test_grouped_indices_out_of_range_stay_inside(dev):
    """Offsets and rows are device data: whatever they hold, reads and writes stay in
    the tensors (values of the rows concerned are not defined)."""
    t, top, e = 60, 2, 4
    routing = moe.sort(router(t, top, e, seed=1).to(dev), e)
    codes, scales = mxfp4.quantize(randn(e, 64, 96, seed=7).to(dev))
    x = randn(t, 96, seed=8, dtype=torch.bfloat16).to(dev).requires_grad_()
    for offsets in ([-5, 1 << 30, 7, -(1 << 31), 120], [0, 300, 20, 90, 50], [120, 0, 0, 0, 0]):
        bad = routing._replace(rows=routing.rows + 1000,
                               offsets=torch.tensor(offsets, dtype=torch.int32, device=dev))
        y = mxfp4.grouped_linear(x, codes, scales, bad, gather=True)
        assert y.shape == (t * top, 64)
        torch.autograd.grad(y, x, torch.ones_like(y))
    torch.cuda.synchronize()


# -------------------------------------------------------------------- graphs
def test_in_a_graph(dev):
    """A captured decode step replays with new inputs, eager work in between."""
    codes, scales = mxfp4.quantize(randn(300, 512, seed=4).to(dev))
    w = mxfp4.quantize(randn(8, 256, 300 // 32 * 32, seed=5).to(dev))
    ids = router(40, 2, 8, seed=3).to(dev)
    x = randn(40, 512, seed=1, dtype=torch.bfloat16).to(dev)

    def step():
        h = mxfp4.linear(x, codes, scales)[:, :288]
        routing = moe.sort(ids, 8)
        return mxfp4.grouped_linear(h, *w, routing, gather=True), routing.position

    for _ in range(2):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, pos = step()
    for seed in (5, 6, 7):
        x.copy_(randn(40, 512, seed=seed, dtype=torch.bfloat16))
        ids.copy_(router(40, 2, 8, seed=seed, dropped=0.1))
        graph.replay()
        torch.cuda.synchronize()
        got, gpos = y.clone(), pos.clone()
        want, wpos = step()
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(gpos, wpos)
