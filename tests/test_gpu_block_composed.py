"""RMS norm, routing and rotary positions together as a block uses them, in graphs, on
several streams and threads, and beyond 2^32 elements."""

import threading

import pytest
import torch

import oracle.block as O
from block_util import U, norm_error, within
from mx_util import DTYPES, big_memory, randn  # noqa: F401
from test_gpu_mx_composed import replays
from test_gpu_rotate_axes import check as check_turned
from xpu_kernels import int8, moe, mxfp4, norm, rope
from xpu_kernels.int8 import _lib as L

pytestmark = pytest.mark.gpu


def test_attention_inputs(dev):
    """The stream's addition, norm and quantization, one projection to q, k and v, the heads'
    norms in its columns and their rotation; each step against 64 bits on its own inputs."""
    b, s, d, h, hk, hd = 2, 37, 512, 4, 2, 64
    x, r = (randn(b, s, d, seed=i, dtype=torch.bfloat16).to(dev) for i in (1, 2))
    g = (1 + 0.2 * randn(d, seed=3)).to(dev)
    qn, kn = ((1 + 0.2 * randn(hd, seed=i)).to(dev) for i in (4, 5))
    w8, ws = int8.prepare_weight(randn((h + 2 * hk) * hd, d, seed=6, scale=0.05).bfloat16().to(dev))
    f = rope.axis_frequencies((8, 12, 12), device=dev)
    pos = torch.stack([torch.arange(s) // 9, torch.arange(s) // 3 % 3, torch.arange(s) % 3]).to(dev)
    codes, scale, stream = norm.rms_norm_int8(x, g, residual=r)
    assert torch.equal(stream, x + r) and codes.shape == x.shape and scale.shape == x.shape[:2]
    qkv = int8.linear_quantized(codes, scale, w8, ws)
    assert qkv.shape == (b, s, (h + 2 * hk) * hd)
    want, _, _ = O.rms_norm(x.cpu(), g.cpu(), 1e-6, r.cpu())
    back = (codes.cpu().double() * scale.cpu().double()[..., None]).unflatten(-1, (-1, 256)) @ O.rotation()
    # each code is off by half a step of its row, and the rotation keeps lengths
    assert ((back.flatten(-2) - want).norm(dim=-1) <= 0.5 * 1.01 * scale.cpu().double() * d ** 0.5).all()
    q = qkv[..., :h * hd].unflatten(-1, (h, hd))
    k = qkv[..., h * hd:(h + hk) * hd].unflatten(-1, (hk, hd))
    nq, nk = norm.rms_norm(q, qn), norm.rms_norm(k, kn)
    for n, t, w in ((nq, q, qn), (nk, k, kn)):
        y, _, _ = O.rms_norm(t.cpu(), w.cpu(), 1e-6)
        within(n, y, (norm_error(hd) + 2 * U) * y.abs())
    tq, tk = rope.rotate_axes(nq, nk, pos, f)
    check_turned(tq, nq.cpu(), pos.cpu(), f, True)
    check_turned(tk, nk.cpu(), pos.cpu(), f, True)


def block(t, d, e, f, dtype, dev):
    up = mxfp4.quantize(randn(e, 2 * f, d, seed=3, scale=0.1).to(dev))
    down = mxfp4.quantize(randn(e, d, f, seed=4, scale=0.1).to(dev))
    x, r = (randn(t, d, seed=i, dtype=dtype).to(dev).requires_grad_() for i in (1, 2))
    g = (1 + 0.2 * randn(d, seed=5)).to(dev).requires_grad_()
    w = randn(e, d, seed=6, scale=0.05).to(dev).requires_grad_()
    bias = (randn(e, seed=7) * 0.02).to(dev)
    return up, down, (x, r, g, w), bias


def experts(up, down, leaves, bias, top, **how):
    x, r, g, w = leaves
    y, h = norm.rms_norm(x, g, residual=r)
    logits = torch.mm(y.float(), w.t())
    ids, weights = moe.route(logits, top, scores="sigmoid", bias=bias, **how)
    return h + moe.ffn(y, ids, weights, up, down), h, y, logits, ids, weights


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,groups", [(3, 1), (70, 4)])
def test_experts_of_a_block(dev, dtype, t, groups):
    """Norm, router, choice, experts and the sum: gradients to the stream, the norm's weight and
    the router's, the same as those of the steps one by one."""
    d, e, f, top = 288, 16, 96, 4
    up, down, leaves, bias = block(t, d, e, f, dtype, dev)
    how = dict(groups=groups, top_groups=max(1, groups // 2), scale=2.0)
    out, h, y, logits, ids, weights = experts(up, down, leaves, bias, top, **how)
    oid, ow = O.route(logits.detach().cpu(), top, "sigmoid", bias.cpu(), **how)
    assert torch.equal(ids.cpu(), oid)
    within(weights, ow, 1e-12 * ow.abs())
    dy = randn(t, d, seed=8, dtype=dtype).to(dev)
    got = torch.autograd.grad(out, leaves, dy)
    x, r, g, w = leaves
    yl, wl, hl = (v.detach().clone().requires_grad_() for v in (y, weights, h))
    dys, dws, dh = torch.autograd.grad(hl + moe.ffn(yl, ids, wl, up, down), (yl, wl, hl), dy)
    ll = logits.detach().clone().requires_grad_()
    dl, = torch.autograd.grad(moe.route(ll, top, scores="sigmoid", bias=bias, **how)[1], ll, dws)
    want = O.route_grad(ll.detach().cpu(), oid, dws.cpu(), "sigmoid", True, 2.0)
    size = 2.0 * ow.abs().sum(-1, keepdim=True) * dws.cpu().double().abs().amax(-1, keepdim=True)
    within(dl, want, 40 * U * size)
    yl = y.detach().clone().requires_grad_()
    wr = w.detach().clone().requires_grad_()
    dy2, dw = torch.autograd.grad(torch.mm(yl.float(), wr.t()), (yl, wr), dl)
    assert torch.equal(got[3], dw)
    xl, rl, gl = (v.detach().clone().requires_grad_() for v in (x, r, g))
    dx, dr, dg = torch.autograd.grad(norm.rms_norm(xl, gl, residual=rl), (xl, rl, gl), (dys + dy2, dh))
    # (the two gradients of y meet in its type, in either order)
    assert torch.equal(got[0], dx) and torch.equal(got[1], dr) and torch.equal(got[2], dg)
    assert all(v.any() for v in got)


# -------------------------------------------------------------------- graphs
@pytest.mark.parametrize("dtype", DTYPES)
def test_experts_of_a_block_in_a_graph(dev, dtype):
    """Captured with its gradients."""
    t, d, e, f, top = 33, 288, 16, 96, 4
    up, down, leaves, bias = block(t, d, e, f, dtype, dev)
    dy = randn(t, d, seed=8, dtype=dtype).to(dev)

    def step():
        out = experts(up, down, leaves, bias, top)
        return (*(v for v in out), *torch.autograd.grad(out[0], leaves, dy))

    def refresh(seed):
        with torch.no_grad():
            for i, v in enumerate(leaves[:2]):
                v.copy_(randn(t, d, seed=seed + i, dtype=dtype))
            leaves[3].copy_(randn(e, d, seed=seed + 2, scale=0.05))
        bias.copy_(randn(e, seed=seed + 3) * 0.02)
        dy.copy_(randn(t, d, seed=seed + 4, dtype=dtype))

    replays(step, refresh)


@pytest.mark.parametrize("native", [True, False])
def test_a_leaf_of_an_eager_graph_is_refused_in_a_capture(dev, monkeypatch, native):
    """While an eager graph of a leaf on the default stream lives, the leaf's gradient belongs to
    that stream, and a captured backward pass, which would make it wait for the capturing one,
    ends the process: the forward call is refused.  Without the graph it is captured."""
    if not native:                                 # every call through the Python code
        check = L.HOST.check_leaves
        monkeypatch.setattr(L, "HOST", type("Declines", (), {
            "__getattr__": lambda self, name: check if name == "check_leaves" else lambda *a: None})())
    f = rope.axis_frequencies((8,), device=dev)
    pos = torch.arange(6, device=dev)[None]
    x, w, r = randn(6, 64, seed=1).to(dev), randn(64, seed=2).to(dev), randn(6, 64, seed=3).to(dev)
    q, k = randn(1, 6, 2, 16, seed=4).to(dev), randn(1, 6, 1, 16, seed=5).to(dev)
    calls = {"norm x": (x, lambda v: norm.rms_norm(v, w)), "norm weight": (w, lambda v: norm.rms_norm(x, v)),
             "view": (x, lambda v: norm.rms_norm(v.view(2, 3, 64)[:1], w)),
             "residual": (r, lambda v: norm.rms_norm(x, w, residual=v)[0]),
             "route": (x, lambda v: moe.route(v, 4)[1]), "q": (q, lambda v: rope.rotate_axes(v, k, pos, f)[0]),
             "k": (k, lambda v: rope.rotate_axes(q, v, pos, f)[1])}
    for name, (v, call) in calls.items():
        leaf = v.clone().requires_grad_()
        call(leaf)                                 # (set up; its graph dies with its result)
        kept = leaf * 2.0
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        refused = False
        with torch.cuda.graph(graph):
            out = x + 1.0
            try:
                call(leaf)
            except RuntimeError as e:
                refused = "still alive" in str(e)
            with torch.no_grad():                  # nothing of a gradient: nothing to refuse
                call(leaf)
        assert refused, name
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, x + 1.0)
        del kept
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call(leaf)
            g, = torch.autograd.grad(y, leaf, y.detach())
        graph.replay()
        torch.cuda.synchronize()
        y2 = call(leaf)
        assert torch.equal(y, y2) and torch.equal(g, torch.autograd.grad(y2, leaf, y2.detach())[0]), name


def test_a_step_whose_warm_up_is_alive_is_captured(dev):
    """The usual order of a captured training step: warmed up on a side stream, whose last
    loss is still there at the capture.  That stream joins the capture and is joined to it."""
    x = randn(9, 64, seed=1).to(dev)
    w, v = (1 + 0.1 * randn(64, seed=2)).to(dev).requires_grad_(), randn(16, 64, seed=3).to(dev).requires_grad_()

    def step():
        y = norm.rms_norm(x, w)
        weights = moe.route(torch.mm(y, v.t()), 4, scores="sigmoid")[1]
        loss = (weights * weights).sum() + (y * y).sum()
        loss.backward()
        return loss

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            w.grad = v.grad = None
            loss = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    w.grad = v.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()                              # (the warm-up's loss lives until this one is there)
    gw, gv = w.grad, v.grad
    for seed in (5, 6, 7):
        x.copy_(randn(9, 64, seed=seed))
        gw.zero_()
        gv.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [gw.clone(), gv.clone()]
        w.grad = v.grad = None
        step()
        torch.cuda.synchronize()
        assert w.grad.any() and v.grad.any()
        assert torch.equal(got[0], w.grad) and torch.equal(got[1], v.grad)


def test_a_leaf_of_a_captured_stream_is_not_refused(dev):
    """Two streams of one capture."""
    x, w = randn(6, 64, seed=1).to(dev).requires_grad_(), randn(64, seed=2).to(dev)
    norm.rms_norm(x, w)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        a = x * 2.0                                # the leaf's gradient belongs to this stream
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b = norm.rms_norm(x, w)
        torch.cuda.current_stream().wait_stream(side)
        out = a + b
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, x * 2.0 + norm.rms_norm(x, w))


@pytest.mark.parametrize("k", [64, 1280, 5120, 33024])
def test_norm_and_rotation_in_a_graph(dev, k):
    m, b, s = 40, 2, 20
    f = rope.axis_frequencies((16, 16), device=dev)
    x, r = (randn(m, k, seed=i, dtype=torch.bfloat16).to(dev).requires_grad_() for i in (1, 2))
    w = (1 + 0.2 * randn(k, seed=3)).to(dev).requires_grad_()
    pos = torch.randint(0, 1000, (2, b, s), device=dev)
    q = randn(b, s, k // 64, 64, seed=4).to(dev).requires_grad_()
    dy, dh = (randn(m, k, seed=i, dtype=torch.bfloat16).to(dev) for i in (5, 6))

    def step():
        y, h = norm.rms_norm(x, w, residual=r)
        oq, _ = rope.rotate_axes(q, None, pos, f)
        with torch.no_grad():
            codes = norm.rms_norm_int8(x, w, residual=r, rotate=k % 256 == 0)
        return (y, h, oq, *codes, *torch.autograd.grad((y, h), (x, w, r), (dy, dh)),
                *torch.autograd.grad(oq, q, q.detach()))

    def refresh(seed):
        with torch.no_grad():
            for i, v in enumerate((x, r)):
                v.copy_(randn(m, k, seed=seed + i, dtype=torch.bfloat16))
            w.copy_(1 + 0.2 * randn(k, seed=seed + 2))
            q.copy_(randn(b, s, k // 64, 64, seed=seed + 3))
        pos.copy_(torch.randint(0, 100000, (2, b, s), generator=torch.Generator().manual_seed(seed)))
        dy.copy_(randn(m, k, seed=seed + 4, dtype=torch.bfloat16))

    replays(step, refresh)


# ------------------------------------------------------------- streams and threads
def test_streams_and_threads(dev):
    """Calls on streams and threads of their own at once give what they give alone."""
    f = rope.axis_frequencies((16, 16), device=dev)

    def work(seed):
        m, k = 300 + 37 * seed, 1280 + 24 * seed
        x, w = randn(m, k, seed=seed).to(dev).requires_grad_(), (1 + 0.2 * randn(k, seed=9)).to(dev).requires_grad_()
        dy = randn(m, k, seed=seed + 1).to(dev)
        lg = randn(m, 64, seed=seed + 2).to(dev).requires_grad_()
        q = randn(1, m, 3, 64, seed=seed + 3).to(dev)
        pos = torch.arange(m, device=dev)[None].expand(2, m)
        torch.cuda.current_stream().synchronize()

        def go():
            y = norm.rms_norm(x, w)
            ids, wt = moe.route(lg, 8, scores="sigmoid", groups=8, top_groups=4)
            return [y, *torch.autograd.grad(y, (x, w), dy), ids, wt, *torch.autograd.grad(wt, lg, wt.detach()),
                    rope.rotate_axes(q, q, pos, f)[0], *norm.rms_norm_int8(x.detach(), w.detach(), rotate=False)]
        return go

    jobs = [work(i) for i in range(4)]
    alone = [[t.clone() for t in j()] for j in jobs]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def run(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(20):
                    got[i] = jobs[i]()
            s.synchronize()
        except Exception as e:                     # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, g in zip(alone, got):
        for u, v in zip(a, g):
            assert torch.equal(u, v)


def test_what_lies_beside_is_left_as_it_was(dev):
    """Results end where they end: odd sizes between other tensors of one buffer."""
    for k in (7, 65, 1001, 5123):
        x = randn(5, k, seed=k, dtype=torch.float16).to(dev)
        before = torch.full((1 << 14,), 7.0, device=dev)
        y = norm.rms_norm(x)
        after = torch.full((1 << 14,), 7.0, device=dev)
        want, _, _ = O.rms_norm(x.cpu(), None, 1e-6)
        within(y, want, (norm_error(k) + 2 * U) * want.abs())
        assert (before == 7.0).all() and (after == 7.0).all()
    # a result whose last row ends in the middle of the library's pieces, seen through the C entry
    lib = L._lib()
    for k in (7, 65, 1001):
        x = randn(3, k, seed=k).to(dev)
        out = torch.full((3 * k + 40,), 7.0, device=dev)
        assert lib.xpuint8_rms_norm_stream(L._stream(dev), x.data_ptr(), 2, k, k, None, 0, 0, 1, None, 0, 1e-6,
                                           None, out.data_ptr(), 3, k) == 0
        assert (out[3 * k:] == 7.0).all() and torch.equal(out[:3 * k].reshape(3, k), norm.rms_norm(x))
        q = torch.full((3 * k + 40,), 7, dtype=torch.int8, device=dev)
        s = torch.full((8,), 7.0, device=dev)
        assert lib.xpuint8_rms_norm_int8_stream(L._stream(dev), x.data_ptr(), 2, k, k, None, 0, 0, 1, None, 0, 1e-6,
                                                None, q.data_ptr(), s.data_ptr(), 0, 3, k) == 0
        assert (q[3 * k:] == 7).all() and (s[3:] == 7.0).all()


# ------------------------------------------------------------------ beyond 2^32 elements
@pytest.mark.parametrize("k", [4096, 66000, 100])
def test_norm_of_many_elements(dev, big_memory, k):
    m = (1 << 32) // k + 5
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=dev)
    rows = torch.tensor([0, 1, m // 2, m - 2, m - 1])
    part = randn(5, k, seed=1, dtype=torch.bfloat16)
    x[rows.to(dev)] = part.to(dev)
    y, h = norm.rms_norm(x, residual=x)
    want, hh, _ = O.rms_norm(part, None, 1e-6, part)
    assert torch.equal(h[rows.to(dev)].cpu(), hh)
    within(y[rows.to(dev)], want, (norm_error(k) + 2 * U) * want.abs())
    assert not y[m // 2 + 1:m // 2 + 9].any()
    del y
    w = torch.ones(k, device=dev, requires_grad=True)
    xg = x.requires_grad_()
    dx, dw = torch.autograd.grad(norm.rms_norm(xg, w), (xg, w), h)
    dy = hh.double()
    odx, odw = O.rms_norm_grad(hh, part, torch.ones(k), 1e-6)
    size = (dy.abs() + dy.norm(dim=-1, keepdim=True)) * (part.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    within(dx[rows.to(dev)], odx, 200 * U * size)
    terms = (dy * part.double()).abs().sum(0) * 3
    within(dw, odw, 200 * U * terms)
    del dx, h
    with torch.no_grad():
        q, s = norm.rms_norm_int8(x, rotate=False)
    code, scale, _ = O.rms_norm_int8(part, None, 1e-6, None, False)
    assert ((q[rows.to(dev)].cpu().double() - code).abs() <= 0.5 + 1e-4).all()
    within(s[rows.to(dev)], scale, scale * (norm_error(k) + 4 * U))


def test_rotation_of_many_elements(dev, big_memory):
    s, h, d = (1 << 32) // (32 * 64) + 3, 32, 64
    f = rope.axis_frequencies((16, 16), device=dev)
    q = torch.zeros(1, s, h, d, dtype=torch.bfloat16, device=dev)
    at = torch.tensor([0, s // 2, s - 1])
    part = randn(1, 3, h, d, seed=1, dtype=torch.bfloat16)
    q[:, at.to(dev)] = part.to(dev)
    pos = torch.arange(s, device=dev, dtype=torch.int32)[None].expand(2, s)
    got, _ = rope.rotate_axes(q, None, pos, f)
    check_turned(got[:, at.to(dev)], part, at[None].expand(2, 3), f, True)
    assert not got[:, s // 2 + 1:s // 2 + 5].any()


def test_route_of_many_elements(dev, big_memory):
    t, e = (1 << 32) // 1024 + 3, 1024
    lg = torch.zeros(t, e, dtype=torch.bfloat16, device=dev)
    at = torch.tensor([0, t // 2, t - 1])
    part = randn(3, e, seed=1, dtype=torch.bfloat16)
    lg[at.to(dev)] = part.to(dev)
    lg.requires_grad_()
    ids, w = moe.route(lg, 4)
    oid, ow = O.route(part, 4)
    assert torch.equal(ids[at.to(dev)].cpu(), oid)
    within(w[at.to(dev)], ow, 1e-12 * ow)
    assert ids[1].tolist() == [0, 1, 2, 3]
    dw = torch.zeros_like(w)
    dw[at.to(dev)] = randn(3, 4, seed=2).to(dev)
    d, = torch.autograd.grad(w, lg, dw)
    within(d[at.to(dev)], O.route_grad(part, oid, dw[at.to(dev)].cpu()), 40 * U * dw.abs().max().item())
    assert not d[1:9].any()
