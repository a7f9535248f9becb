"""RMS norm with the residual's addition, its gradient and its int8 form on the device
against the 64-bit oracle."""

import pytest
import torch

import oracle.block as O
from block_util import U, chain, norm_error, within
from mx_util import DTYPES, randn
from xpu_kernels import int8, norm

pytestmark = pytest.mark.gpu

# rows a lane, a wave, a block and many; lengths at the ends of each kernel's range
SHAPES = [(1, 1), (3, 7), (65, 8), (33, 64), (17, 65), (40, 100), (9, 128), (8, 255), (5, 512),
          (3, 513), (2, 1000), (7, 1280), (5, 1537), (3, 2048), (2, 2049), (4, 4096), (3, 5120),
          (2, 6151), (2, 8192), (3, 8193), (2, 16384), (1, 16385), (2, 32768), (2, 32769), (1, 70001)]


def stream(m, k, dtype, seed):
    x = randn(m, k, seed=seed)
    x[:, ::97] *= 30.0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", SHAPES)
def test_forward(dev, dtype, m, k):
    x, r = stream(m, k, dtype, 1), stream(m, k, dtype, 2)
    for wt, res in ((None, None), (dtype, r), (torch.float32, None), (torch.float16, r)):
        w = None if wt is None else (1 + 0.2 * randn(k, seed=3)).to(wt)
        got = norm.rms_norm(x.to(dev), None if w is None else w.to(dev), 1e-5,
                            residual=None if res is None else res.to(dev))
        want, h, _ = O.rms_norm(x, w, 1e-5, res)
        if res is not None:
            got, gh = got
            assert torch.equal(gh.cpu(), h)
        assert got.dtype == dtype
        within(got, want, (norm_error(k) + 2 * U) * want.abs())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", SHAPES + [(700, 64), (600, 1280), (1500, 4096), (2, 0 + 24)])
def test_gradient(dev, dtype, m, k):
    x, r = stream(m, k, dtype, 1), stream(m, k, dtype, 2)
    dy, dh = randn(m, k, seed=4, dtype=dtype), randn(m, k, seed=5, dtype=dtype)
    for wt, res in ((dtype, r), (torch.float32, None)):
        w = (1 + 0.2 * randn(k, seed=3)).to(wt)
        leaves = [t.to(dev).requires_grad_() for t in ((x, w) if res is None else (x, w, res))]
        if res is None:
            out, grads = (norm.rms_norm(*leaves, 1e-5),), (dy.to(dev),)
        else:
            out = norm.rms_norm(leaves[0], leaves[1], 1e-5, residual=leaves[2])
            grads = (dy.to(dev), dh.to(dev))
        got = torch.autograd.grad(out, leaves, grads)
        _, h, rr = O.rms_norm(x, w, 1e-5, res)
        dx, dw = O.rms_norm_grad(dy, h, w, 1e-5, None if res is None else dh)
        # r g, h r^3 mean(g h): r's error once and three times, the sum along h's, a few products
        g, hd = (dy.double() * w.double()).abs(), h.double().abs()
        e = norm_error(k)
        error = rr * g * (e + 4 * U) + hd * rr ** 3 * (g * hd).mean(-1, keepdim=True) * (
            3 * e + (chain(k) + 8) * U)
        if res is not None:
            error = error + 2 * U * (dh.double().abs() + dx.abs())
            assert torch.equal(got[0], got[2])
        within(got[0], dx, error)
        # a row's term to r's error, then the additions: rows of a block, 32 groups of it, up to
        # 512 blocks in 32 slices
        terms = (dy.double() * h.double() * rr).abs().sum(0)
        within(got[1], dw, terms * (e + (2 + -(-m // 512) + 32 + 16 + 32) * U))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [1e-15, 1e15])
@pytest.mark.parametrize("k", [7, 100, 1280, 5120, 16390])
def test_gradient_of_rows_whose_cube_is_out_of_range(dev, dtype, size, k):
    """r ** 3 is 10 ** 45 or 10 ** -45; what the formula makes of it is not."""
    x, w = (randn(5, k, seed=1) * size).to(dtype), (1 + 0.2 * randn(k, seed=3)).to(dtype)
    dy = (randn(5, k, seed=4) + 0.5 * torch.sign(x.float())).to(dtype)
    leaves = [x.to(dev).requires_grad_(), w.to(dev).requires_grad_()]
    got = torch.autograd.grad(norm.rms_norm(*leaves, 0.0), leaves, dy.to(dev))
    _, h, rr = O.rms_norm(x, w, 0.0)
    dx, dw = O.rms_norm_grad(dy, h, w, 0.0)
    g, hd = (dy.double() * w.double()).abs(), h.double().abs()
    e = norm_error(k)
    within(got[0], dx, rr * g * (e + 4 * U) + hd * rr ** 3 * (g * hd).mean(-1, keepdim=True) * (
        3 * e + (chain(k) + 8) * U))
    within(got[1], dw, (dy.double() * h.double() * rr).abs().sum(0) * (e + 90 * U))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,rotate", [(m, k, rotate) for m, k in [
    (1, 256), (3, 512), (5, 768), (7, 1280), (2, 2304), (4, 4096), (3, 5120), (2, 16384), (2, 16640),
    (1, 66560), (2, 17), (3, 1001), (2, 8200), (1, 33000), (70, 256)]
    for rotate in ([True, False] if k % 256 == 0 else [False])])
def test_int8(dev, dtype, m, k, rotate):
    x, r = stream(m, k, dtype, 1), stream(m, k, dtype, 2)
    for wt, res in ((None, None), (dtype, r), (torch.float32, r)):
        w = None if wt is None else (1 + 0.2 * randn(k, seed=3)).to(wt)
        got = norm.rms_norm_int8(x.to(dev), None if w is None else w.to(dev), 1e-5,
                                 residual=None if res is None else res.to(dev), rotate=rotate)
        code, scale, h = O.rms_norm_int8(x, w, 1e-5, res, rotate)
        q, s = got[0].cpu().double(), got[1]
        if res is not None:
            assert torch.equal(got[2].cpu(), h)
        # v's product (one rounding), the rotation's 12 additions of the group's magnitudes,
        # the maximum's the same, the quotient and the product with it
        v = (h.double() * (1.0 if w is None else w.double())).abs()
        size = v if not rotate else v.unflatten(-1, (-1, 256)).sum(-1, keepdim=True).expand(
            -1, -1, 256).flatten(-2) / 16
        m_ = (scale / O.rms_norm(x, w, 1e-5, res)[2][..., 0] * 127)[..., None]
        error = (13 if rotate else 1) * U * size / m_ * 127
        most = error.amax(-1, keepdim=True)
        off = (q - code).abs() - 0.5 - error - code.abs() * (most / 127 + 3 * U)
        assert off.max() <= 0, float(off.max())
        assert q.abs().max() <= 127
        within(s, scale, scale * (norm_error(k) + most[..., 0] / 127 + 3 * U))


def test_int8_of_zeros_and_tiny_rows(dev):
    x = torch.zeros(4, 512)
    x[1] = 1e-30
    x[2, 5] = 1e-38
    x[3, 7] = 3.0
    for rotate in (True, False):
        q, s = norm.rms_norm_int8(x.to(dev), None, 1e-6, rotate=rotate)
        code, scale, _ = O.rms_norm_int8(x, None, 1e-6, None, rotate)
        assert (q.cpu().double() - code).abs().max() <= 0.5 + 1e-4
        assert torch.allclose(s.cpu().double(), scale, rtol=1e-5, atol=0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("k", [64, 1280, 4096, 33024])
def test_not_finite(dev, dtype, value, k):
    """The row with the value is NaN where the formula's is, the others as they were."""
    x = stream(5, k, dtype, 1)
    clean = norm.rms_norm(x.to(dev), eps=1e-6)
    q0, s0 = norm.rms_norm_int8(x.to(dev), rotate=False)
    x[2, k // 2] = value
    y = norm.rms_norm(x.to(dev), eps=1e-6).cpu()
    rows = [0, 1, 3, 4]
    assert torch.equal(y[rows], clean.cpu()[rows])
    want = torch.full((k,), float("nan")) if value != value else torch.zeros(k)
    want[k // 2] = float("nan")
    assert torch.equal(y[2].float().nan_to_num(7.0), want.nan_to_num(7.0))
    for rotate in ([False, True] if k % 256 == 0 else [False]):
        q, s = norm.rms_norm_int8(x.to(dev), rotate=rotate)
        assert s[2].isnan() and not s[rows].isnan().any()
        if not rotate:
            assert torch.equal(q[rows], q0[rows]) and torch.equal(s[rows], s0[rows])


def test_extremes(dev):
    """Squares beyond fp32's range make a row zeros; the smallest ones eps decides."""
    x = torch.tensor([[3e38, 1.0, -2e38, 0.0], [1e-30, 2e-30, 0.0, 1e-38]])
    y = norm.rms_norm(x.to(dev), eps=1e-6).cpu()
    assert torch.equal(y[0].abs(), torch.zeros(4))
    within(y[1], O.rms_norm(x[1:], None, 1e-6)[0][0], 64 * U * y[1].double().abs())
    y = norm.rms_norm(torch.zeros(2, 40, device=dev), eps=0.0)
    assert y.isnan().all()                                 # 0 / 0
    h = torch.full((1, 300), 60000.0, dtype=torch.float16)
    y, hh = norm.rms_norm(h.to(dev), eps=0.0, residual=h.to(dev))
    assert (hh == float("inf")).all() and y.isnan().all()  # inf / inf


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dev, dtype):
    """Column slices, transposed and expanded rows, odd starts, 1-D and empty inputs."""
    base = stream(40, 1400, dtype, 1).to(dev)
    w = (1 + 0.2 * randn(1400, seed=3)).to(dev)
    for x in (base[:, 3:1284], base[::2, :1280], base.t()[:1400], base[:1].expand(6, 1400),
              base[:, 1:2], base.reshape(8, 5, 1400)[:, 2], base[0], base.reshape(4, 10, 1400)):
        k = x.shape[-1]
        want = norm.rms_norm(x.contiguous().clone(), w[:k].clone(), 1e-5)
        assert torch.equal(norm.rms_norm(x, w[:k], 1e-5), want)
        y, h = norm.rms_norm(x, w[:k], 1e-5, residual=x)
        y2, h2 = norm.rms_norm(x.contiguous(), w[:k].clone(), 1e-5, residual=x.contiguous())
        assert torch.equal(h, x + x) and torch.equal(y, y2) and torch.equal(h, h2)
        q, s, h3 = norm.rms_norm_int8(x, w[:k], 1e-5, residual=x, rotate=False)
        q2, s2 = norm.rms_norm_int8(h2, w[:k], 1e-5, rotate=False)
        assert torch.equal(q, q2) and torch.equal(s, s2) and torch.equal(h3, h2)
        assert q.shape == x.shape and s.shape == x.shape[:-1]
        xg = x.detach().clone().requires_grad_()
        xs = torch.as_strided(x.detach(), x.shape, x.stride(), x.storage_offset()).requires_grad_()
        dy = randn(*x.shape, seed=9, dtype=dtype).to(dev)
        wide = torch.zeros(*x.shape[:-1], k + 3, dtype=dtype, device=dev)
        wide[..., 1:k + 1] = dy
        a, = torch.autograd.grad(norm.rms_norm(xg, w[:k]), xg, dy)
        b, = torch.autograd.grad(norm.rms_norm(xs, w[:k]), xs, wide[..., 1:k + 1])
        assert torch.equal(a, b)
    # heads in the columns of one projection, and layouts that are neither rows nor runs
    qkv = stream(12, 3 * 4 * 72 + 5, dtype, 2).to(dev).reshape(3, 4, -1)
    wq = (1 + 0.2 * randn(72, seed=3)).to(dev)
    q, k = (qkv[..., i * 288 + 1:(i + 1) * 288 + 1].unflatten(-1, (4, 72)) for i in (0, 1))
    for x, r in ((q, k), (q, k.contiguous()), (q.contiguous(), k), (q.transpose(1, 2), k.transpose(1, 2)),
                 (q[:, ::2], k[:, 1::2]), (q[:, :, ::2], k[:, :, ::2]), (q, k.transpose(0, 1).contiguous().transpose(0, 1)),
                 (q[:1], k[:1]), (q[:, :1], k[:, :1]), (q[:, :, :1], k[:, :, :1]),
                 (q[:1].expand(3, 4, 4, 72), k[:, :1].expand(3, 4, 4, 72)), (q[:, :, :1].expand(3, 4, 4, 72), k)):
        xc, rc = x.contiguous(), r.contiguous()
        y, h = norm.rms_norm(x, wq, residual=r)
        yc, hc = norm.rms_norm(xc, wq, residual=rc)
        assert torch.equal(y, yc) and torch.equal(h, hc) and torch.equal(norm.rms_norm(x, wq), norm.rms_norm(xc, wq))
        for a, b in zip(norm.rms_norm_int8(x, wq, residual=r, rotate=False),
                        norm.rms_norm_int8(xc, wq, residual=rc, rotate=False)):
            assert torch.equal(a, b)
        for dy in (r, rc):
            xs, xg = x.detach().requires_grad_(), xc.clone().requires_grad_()
            a, = torch.autograd.grad(norm.rms_norm(xs, wq), xs, dy)
            b, = torch.autograd.grad(norm.rms_norm(xg, wq), xg, rc)
            assert torch.equal(a, b)
            a = torch.autograd.grad(norm.rms_norm(xs, wq, residual=r), xs, (dy, x))
            b = torch.autograd.grad(norm.rms_norm(xg, wq, residual=rc), xg, (rc, xc))
            assert torch.equal(a[0], b[0])
    empty = torch.empty(0, 1280, dtype=dtype, device=dev)
    assert norm.rms_norm(empty, w[:1280]).shape == (0, 1280)
    q, s, h = norm.rms_norm_int8(empty, w[:1280], residual=empty)
    assert q.shape == h.shape == (0, 1280) and s.shape == (0,)
    e, wg = empty.clone().requires_grad_(), w[:1280].clone().requires_grad_()
    de, dw = torch.autograd.grad(norm.rms_norm(e, wg), (e, wg), empty)
    assert de.shape == (0, 1280) and torch.equal(dw, torch.zeros_like(wg))


def test_gradients_of_one_output_and_one_input(dev):
    x, r, w = (randn(6, 320, seed=i).to(dev) for i in (1, 2, 3))
    w = w[0].clone()
    dy, dh = randn(6, 320, seed=4).to(dev), randn(6, 320, seed=5).to(dev)
    leaves = [t.clone().requires_grad_() for t in (x, w, r)]
    y, h = norm.rms_norm(leaves[0], leaves[1], residual=leaves[2])
    full = torch.autograd.grad((y, h), leaves, (dy, dh), retain_graph=True)
    only_y = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    only_h = torch.autograd.grad(h, leaves, dh, retain_graph=True)
    assert torch.equal(only_h[0], dh) and torch.equal(only_h[2], dh)
    assert torch.equal(only_h[1], torch.zeros_like(w))
    assert torch.allclose(only_y[0] + dh, full[0], rtol=1e-6, atol=1e-6)
    assert torch.equal(only_y[1], full[1])
    for i in range(3):
        some = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
        out = norm.rms_norm(some[0], some[1], residual=some[2])
        g, = torch.autograd.grad(out[:1] if i == 1 else out, some[i], (dy,) if i == 1 else (dy, dh))
        assert torch.equal(g, full[i])
    # the sum of a gradient that is one number everywhere, and the same tensor for both
    xg = x.clone().requires_grad_()
    y, h = norm.rms_norm(xg, w, residual=xg)
    g, = torch.autograd.grad(y.sum() + h.sum(), xg)
    a, _ = O.rms_norm_grad(torch.ones(6, 320), h.cpu(), w.cpu(), 1e-6, torch.ones(6, 320))
    within(g, 2 * a, 64 * U * (2 * a.abs() + 8))


def test_gradient_against_differences(dev):
    """The gradient is that of what the kernels compute: central differences in fp32."""
    x, w = randn(2, 70, seed=1).to(dev), randn(70, seed=2).to(dev)
    dy = randn(2, 70, seed=3).to(dev)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(norm.rms_norm(xg, wg), (xg, wg), dy)
    step = 2.0 ** -7
    for i in range(0, 70, 9):
        e = torch.zeros_like(x)
        e[1, i] = step
        d = ((norm.rms_norm(x + e, w) - norm.rms_norm(x - e, w)).double() * dy.double()).sum() / (2 * step)
        # the third derivative's term, step^2 / 6, and the roundings, 2^-22 / step
        assert abs(d - dx[1, i]) < 2e-3
        e = torch.zeros_like(w)
        e[i] = step
        d = ((norm.rms_norm(x, w + e) - norm.rms_norm(x, w - e)).double() * dy.double()).sum() / (2 * step)
        assert abs(d - dw[i]) < 2e-3


@pytest.mark.parametrize("m", [5, 300])
def test_feeds_the_int8_linear(dev, m):
    """Norm, codes and the product against the same in 64 bits on the codes."""
    k, n = 1280, 320
    x, r = (stream(m, k, torch.bfloat16, i).to(dev) for i in (1, 2))
    w = (1 + 0.2 * randn(k, seed=3)).to(dev)
    w8, ws = int8.prepare_weight(randn(n, k, seed=4, scale=0.02).bfloat16().to(dev))
    bias = randn(n, seed=5, dtype=torch.bfloat16).to(dev)
    q, s, h = norm.rms_norm_int8(x, w, residual=r)
    y = int8.linear_quantized(q, s, w8, ws, bias)
    acc = q.cpu().double() @ w8.cpu().double().t()
    scale = (ws[None] * s[:, None]).cpu().double()
    want = acc * scale + bias.cpu().double()
    within(y, want, 3 * U * (acc.abs() * scale + bias.cpu().double().abs()))
    # and near the linear of the rounded norm: two quantizations of it, each off by half a
    # step of its row (1/254 of its largest value) and of independent signs
    near = int8.linear(norm.rms_norm(x, w, residual=r)[0], w8, ws, bias)
    assert (near.float() - y.float()).norm() < 0.02 * y.float().norm()
    # rows as they are against a weight as it is
    wq, wsr = int8.quantize_row(randn(n, k, seed=4, scale=0.02).bfloat16().to(dev))
    q, s, _ = norm.rms_norm_int8(x, w, residual=r, rotate=False)
    acc = q.cpu().double() @ wq.cpu().double().t()
    scale = (wsr[None] * s[:, None]).cpu().double()
    within(int8.linear_quantized(q, s, wq, wsr), acc * scale, 2 * U * acc.abs() * scale)


@pytest.mark.parametrize("m,n,k", [(1, 16, 16), (5, 48, 80), (17, 16, 2064), (64, 320, 1296), (257, 1040, 528),
                                   (3, 4112, 4096), (1000, 64, 272)])
def test_linear_of_quantized_rows(dev, m, n, k):
    """Multiples of 16, any strides, scalar scales, no rows."""
    g = torch.Generator().manual_seed(m)
    q, w8 = (torch.randint(-127, 128, (r, k), generator=g, dtype=torch.int8) for r in (m, n))
    s, ws, b = (torch.rand(r, generator=g) + 0.5 for r in (m, n, n))
    acc = q.double() @ w8.double().t()
    for bias in (None, b, b.bfloat16()):
        want = acc * (ws[None] * s[:, None]).double() + (0 if bias is None else bias.double())
        error = 3 * U * (acc.abs() * (ws[None] * s[:, None]).double() + (0 if bias is None else bias.double().abs()))
        bd = None if bias is None else bias.to(dev)
        y = int8.linear_quantized(q.to(dev), s.to(dev), w8.to(dev), ws.to(dev), bd)
        within(y, want, error)
        wide = torch.zeros(m, k + 16, dtype=torch.int8, device=dev)
        wide[:, 3:k + 3] = q.to(dev)
        assert torch.equal(int8.linear_quantized(wide[:, 3:k + 3], s.to(dev)[:, None], w8.to(dev).t().contiguous().t(),
                                                 ws.to(dev)[:, None], bd), y)
        assert torch.equal(int8.linear_quantized(q.to(dev)[None], s.to(dev)[None], w8.to(dev), ws.to(dev), bd), y[None])
    one = int8.linear_quantized(q.to(dev), s.to(dev), w8.to(dev), 0.25)
    within(one, acc * 0.25 * s[:, None].double(), 3 * U * acc.abs() * s[:, None].double())
    assert int8.linear_quantized(q.to(dev)[:0], s.to(dev)[:0], w8.to(dev), 0.25).shape == (0, n)
    with pytest.raises(RuntimeError, match="no gradient"):
        int8.linear_quantized(q.to(dev), s.to(dev).requires_grad_(), w8.to(dev), 0.25)
