"""Captured backward passes beside eager graphs of the default stream: refused where the pass
would go on to one, by whatever way, and nowhere else."""

import pytest
import torch

from mx_util import randn
from xpu_kernels import int8, moe, mxfp4, norm, rope
from xpu_kernels.int8 import _lib as L

pytestmark = pytest.mark.gpu


def calls(dev):
    """Each operator as a function of one tensor [6, 64]"""
    f = rope.axis_frequencies((8,), device=dev)
    pos, w = torch.arange(6, device=dev)[None], randn(64, seed=2).to(dev)
    x, ones = randn(6, 64, seed=5).to(dev), torch.ones(6, 1, device=dev)
    codes = mxfp4.quantize(randn(32, 64, seed=3).to(dev))
    many = mxfp4.quantize(randn(4, 32, 64, seed=4).to(dev))
    routing = moe.sort(torch.tensor([[0], [2], [1], [3], [0], [2]], dtype=torch.int32, device=dev), 4)
    w8, ws = int8.prepare_weight(randn(32, 256, seed=6).bfloat16().to(dev))
    return {"norm": lambda v: norm.rms_norm(v, w), "residual": lambda v: norm.rms_norm(v, w, residual=v * 2.0)[0],
            "weight": lambda v: norm.rms_norm(x, v[0] * w), "route": lambda v: moe.route(v, 4)[1],
            "rope": lambda v: rope.rotate_axes(v.view(1, 6, 2, 32), None, pos, f)[0],
            "linear": lambda v: mxfp4.linear(v, *codes),
            "grouped": lambda v: mxfp4.grouped_linear(v, *many, routing, gather=True),
            "dispatch": lambda v: moe.dispatch(v, routing), "combine": lambda v: moe.combine(v, routing, ones),
            "int8": lambda v: int8.int8_linear(v.reshape(1, 384)[:, :256].bfloat16(), w8, ws, mode="int8")}


class Declines:
    """The native host path without its calls, so that those go through Python."""

    def __init__(self, host):
        self.host = host

    def __getattr__(self, name):
        return getattr(self.host, name) if name.startswith("check_") else lambda *a: None


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("way", ["two inputs", "far", "an eager node"])
@pytest.mark.parametrize("name", ["norm", "residual", "weight", "route", "rope", "linear", "grouped", "dispatch",
                                  "combine", "int8"])
def test_a_leaf_behind_other_nodes(dev, monkeypatch, name, way, native):
    """The leaf's gradient, or a node on the way to it, belongs to the default stream; the forward
    call cannot tell or is not asked, the backward pass is refused before it goes there."""
    if not native:
        monkeypatch.setattr(L, "HOST", Declines(L.HOST))
    call = calls(dev)[name]
    leaf, other = randn(6, 64, seed=1).to(dev).requires_grad_(), randn(6, 64, seed=7).to(dev).requires_grad_()
    kept = leaf * 2.0                              # an eager graph of the leaf, alive
    eager = leaf * other if way == "an eager node" else None

    def inner():
        if way == "an eager node":
            return eager + other                   # (two inputs: not followed by the forward call)
        if way == "two inputs":
            return leaf * other
        v = leaf
        for _ in range(20):
            v = v + 1.0
        return v

    call(leaf.detach())                            # (set up)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mid = inner()
        out = call(mid)                            # no backward pass: captured
        with pytest.raises(RuntimeError, match="still alive"):
            out.backward(out.detach())
        # a pass that stops before the leaf is not refused
        g, = torch.autograd.grad(call(mid), mid, out.detach())
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        want = call(inner())
        assert torch.equal(out, want)
        m = inner()
        assert torch.equal(g, torch.autograd.grad(call(m), m, out.detach())[0])
    assert kept.grad_fn is not None and leaf.grad is None


@pytest.mark.parametrize("native", [True, False])
def test_a_step_without_an_eager_graph_is_captured(dev, monkeypatch, native):
    """The same calls with two inputs, once no graph of the leaves lives."""
    if not native:
        monkeypatch.setattr(L, "HOST", Declines(L.HOST))
    for name, call in calls(dev).items():
        leaf, other = randn(6, 64, seed=1).to(dev).requires_grad_(), randn(6, 64, seed=7).to(dev).requires_grad_()
        call(leaf * other)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(leaf * other)
            got = torch.autograd.grad(out, (leaf, other), out.detach())
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            y = call(leaf * other)
            want = torch.autograd.grad(y, (leaf, other), y.detach())
            assert torch.equal(out, y) and all(torch.equal(a, b) for a, b in zip(got, want)), name


def test_side_streams_without_a_capture(dev):
    """Eager passes on another stream go to graphs of the default stream as before."""
    for name, call in calls(dev).items():
        leaf, other = randn(6, 64, seed=1).to(dev).requires_grad_(), randn(6, 64, seed=7).to(dev)
        kept = leaf * 2.0
        y = call(leaf * other)
        want, = torch.autograd.grad(y, leaf, y.detach())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y = call(leaf * other)
            got, = torch.autograd.grad(y, leaf, y.detach())
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want), name
        del kept
