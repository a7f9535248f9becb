"""Rotary positions on several axes on the device against the 64-bit oracle."""

import pytest
import torch

import oracle.block as O
from block_util import U, within
from mx_util import DTYPES, randn
from xpu_kernels import rope

pytestmark = pytest.mark.gpu


def positions_of(axes, b, s, kind, seed=3, most=3000):
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(0, most, (axes, b, s) if b else (axes, s), generator=g)
    return p.to(kind) if kind != torch.float32 else p.float() / 3


def check(got, x, positions, f, split, inverse=False):
    want = O.rotate_axes(x, positions, f.inv_freq.cpu(), f.axis.cpu(), split, inverse)
    # cosine and sine to 4 units (the part of a turn's rounding, 2^-26 turns, and 2 of the
    # functions), two products and a sum of |a| + |b|; the angle itself in 64 bits
    n = f.axis.numel()
    size = x.double().abs()
    turned = size[..., :2 * n].unflatten(-1, (2, n) if split else (n, 2))
    both = turned.sum(-2 if split else -1, keepdim=True).expand_as(turned).flatten(-2)
    error = torch.cat([8 * U * both, torch.zeros_like(size[..., 2 * n:])], -1)
    within(got, want, error)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("b,s,hq,hk,d,sections,kind", [
    (1, 1, 1, 1, 2, (1,), torch.int32), (1, 1, 32, 8, 128, (16, 24, 24), torch.int32),
    (2, 33, 4, 2, 64, (8, 12, 12), torch.int64), (3, 5, 5, 1, 80, (8, 12, 12), torch.float32),
    (2, 7, 3, 3, 50, (5, 3, 2), torch.int32), (1, 130, 2, 1, 33, (7,), torch.int64),
    (2, 3, 1, 2, 19, (1, 0, 4), torch.int32), (5, 1, 7, 7, 256, (128,), torch.int32),
    (1, 9, 2, 2, 1030, (200, 300, 12), torch.int32), (4, 6, 12, 4, 96, (10, 10, 10, 10), torch.int64),
    (1, 2, 70, 70, 4, (1, 1), torch.int32), (1, 3, 1, 1, 4096, (512,), torch.int32),
    (2, 2, 2, 1, 4096, (1,), torch.int32), (1, 3, 2, 2, 4095, (3, 6), torch.int64),
    (3, 1500, 1, 1, 24, (8, 2), torch.int32), (2, 2111, 3, 2, 10, (4,), torch.int32)])
def test_forward_and_gradient(dev, dtype, split, b, s, hq, hk, d, sections, kind):
    q, k = randn(b, s, hq, d, seed=1, dtype=dtype), randn(b, s, hk, d, seed=2, dtype=dtype)
    dq, dk = randn(b, s, hq, d, seed=4, dtype=dtype), randn(b, s, hk, d, seed=5, dtype=dtype)
    for shared, whole in ((True, True), (False, False)):
        f = rope.axis_frequencies(sections, shared=shared, interleaved=not shared, device=dev)
        p = positions_of(len(sections), b if whole else 0, s, kind)
        qg, kg = q.to(dev).requires_grad_(), k.to(dev).requires_grad_()
        oq, ok = rope.rotate_axes(qg, kg, p.to(dev), f, split_half=split)
        assert oq.dtype == ok.dtype == dtype
        check(oq, q, p, f, split)
        check(ok, k, p, f, split)
        gq, gk = torch.autograd.grad((oq, ok), (qg, kg), (dq.to(dev), dk.to(dev)))
        check(gq, dq, p, f, split, inverse=True)
        check(gk, dk, p, f, split, inverse=True)
        with torch.no_grad():
            alone, none = rope.rotate_axes(qg, None, p.to(dev), f, split_half=split)
            assert none is None and torch.equal(alone, oq)


def test_frequencies():
    f = rope.axis_frequencies((2, 3, 1), 100.0, device="cpu")
    assert f.axis.tolist() == [0, 0, 1, 1, 1, 2]
    assert torch.allclose(f.inv_freq, 100.0 ** (-torch.arange(6).double() / 6), rtol=1e-15)
    f = rope.axis_frequencies((2, 3, 1), 100.0, shared=False, device="cpu")
    assert torch.allclose(f.inv_freq, 100.0 ** -torch.tensor([0, 1 / 2, 0, 1 / 3, 2 / 3, 0]).double(),
                          rtol=1e-7)
    f = rope.axis_frequencies((2, 3, 1), interleaved=True, device="cpu")
    assert f.axis.tolist() == [0, 1, 2, 0, 1, 1]


@pytest.mark.parametrize("kind", [torch.int32, torch.int64, torch.float32])
def test_far_positions(dev, kind):
    """Positions of a long context and beyond, negative ones and fractions."""
    x = randn(1, 12, 2, 64, seed=1)
    p = torch.tensor([[0, 1, -1, 4095, 131071, 1 << 20, 10 ** 7, -(10 ** 7), 1 << 24, (1 << 30) + 64,
                       -(1 << 30), (1 << 31) - 128]])
    p = p.to(kind) if kind != torch.float32 else p.float() + 0.5
    f = rope.axis_frequencies((32,), device=dev)
    got, _ = rope.rotate_axes(x.to(dev), None, p.to(dev), f)
    want = O.rotate_axes(x, p, f.inv_freq.cpu(), f.axis.cpu())
    # the angle in 64 bits: 3 roundings of up to 2^31 radians in 1 / 2^53 each, in both
    within(got, want, (8 * U + 6 * 2.0 ** -22) * x.abs().amax() * 2)


def test_axes_out_of_range_do_not_turn(dev):
    x = randn(1, 3, 2, 16, seed=1)
    f = rope.AxisFrequencies(torch.ones(6, dtype=torch.float64, device=dev),
                             torch.tensor([0, -1, 1, 2, 1 << 30, -(1 << 31)], dtype=torch.int32,
                                          device=dev))
    p = torch.tensor([[1, 2, 3], [4, 5, 6]])
    got, _ = rope.rotate_axes(x.to(dev), None, p.to(dev), f)
    check(got, x, p, f, True)
    for j in (1, 3, 4, 5):
        assert torch.equal(got.cpu()[..., [j, j + 6]], x[..., [j, j + 6]])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("split", [True, False])
def test_layouts(dev, dtype, split):
    """Columns of one projection, heads before positions, expanded and reversed-stride heads,
    odd starts: results of the contiguous ones, in the same layout where it is dense."""
    b, s, h, d = 2, 9, 4, 48
    f = rope.axis_frequencies((8, 9, 3), device=dev)
    p = positions_of(3, b, s, torch.int32).to(dev)
    qkv = randn(b, s, 3 * h * d + 5, seed=1, dtype=dtype).to(dev)
    base = randn(b, h, s, d, seed=2, dtype=dtype).to(dev)
    views = [(qkv[..., 1:h * d + 1].unflatten(-1, (h, d)), qkv[..., h * d + 1:2 * h * d + 1].unflatten(-1, (h, d))),
             (base.transpose(1, 2), base[:, :2].transpose(1, 2)),
             (base[:, :1].transpose(1, 2).expand(b, s, h, d), base[:, 1:3].transpose(1, 2)),
             (randn(b, s, d, h, seed=3, dtype=dtype).to(dev).transpose(2, 3), base.transpose(1, 2)[:, :, ::2]),
             (randn(s, b, h, d, seed=4, dtype=dtype).to(dev).transpose(0, 1), base.transpose(1, 2)[..., :, :])]
    for q, k in views:
        wq, wk = rope.rotate_axes(q.contiguous(), k.contiguous(), p, f, split_half=split)
        for pos in (p, p.long(), p.transpose(1, 2).contiguous().transpose(1, 2)):
            gq, gk = rope.rotate_axes(q, k, pos, f, split_half=split)
            assert torch.equal(gq, wq) and torch.equal(gk, wk)
        qg, kg = q.detach().requires_grad_(), k.detach().requires_grad_()
        out = rope.rotate_axes(qg, kg, p, f, split_half=split)
        dq, dk = torch.autograd.grad(out, (qg, kg), (q, k))
        back = rope._turn(q.contiguous(), k.contiguous(), p, f, True, split)
        assert torch.equal(dq, back[0]) and torch.equal(dk, back[1])
    got, _ = rope.rotate_axes(base.transpose(1, 2), None, p, f)
    assert got.stride() == base.transpose(1, 2).stride()
    empty = torch.empty(2, 0, 3, 48, dtype=dtype, device=dev)
    assert rope.rotate_axes(empty, None, p[..., :0], f)[0].shape == (2, 0, 3, 48)


def test_gradients_of_one_result(dev):
    f = rope.axis_frequencies((8, 8), device=dev)
    p = positions_of(2, 1, 6, torch.int32).to(dev)
    q, k = (randn(1, 6, n, 32, seed=n).to(dev).requires_grad_() for n in (2, 1))
    oq, ok = rope.rotate_axes(q, k, p, f)
    gq, gk = torch.autograd.grad(oq.sum() + 3 * ok.sum(), (q, k), retain_graph=True)
    a, = torch.autograd.grad(oq.sum(), q, retain_graph=True)
    b, = torch.autograd.grad(ok.sum(), k, retain_graph=True)
    assert torch.equal(a, gq) and torch.allclose(3 * b, gk)
    out, _ = rope.rotate_axes(q.detach(), k, p, f)
    assert out.requires_grad                               # (both are results of one call)
    g, = torch.autograd.grad(rope.rotate_axes(q.detach(), k, p, f)[1].sum(), k)
    assert torch.equal(g, b)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(oq.sum(), q, create_graph=True)[0].sum(), q)


def test_no_state_between_calls(dev):
    """Other positions in the same buffer are other angles."""
    f = rope.axis_frequencies((8,), device=dev)
    x = randn(1, 4, 2, 16, seed=1).to(dev)
    p = torch.arange(4, device=dev)[None]
    a, _ = rope.rotate_axes(x, None, p, f)
    p += 1
    b, _ = rope.rotate_axes(x, None, p, f)
    assert not torch.equal(a, b)
    check(b, x.cpu(), p.cpu(), f, True)
