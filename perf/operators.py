"""Performance cases of the 4-bit mixture-of-experts operators: MXFP4
quantization and its reading back, the MXFP4 linear with its gradient, tokens
sorted by expert and back with their gradients, and the experts' products.

``listed()`` are fixed cases, ``draw()`` gives more of the same ranges,
``prepare()`` makes what a program holds before the call and ``run()`` is one
pass: the plain form in elementary torch operations in 32 bits, or with ``own``
the library's calls.  ``exact()`` restates each operator in 64 bits.

A prepared MXFP4 weight is ``codes`` uint8 [.., N, K/2] (element 2i in the low
half of byte i) and ``scales`` uint8 [.., N, 16 ceil(K/512)] (the power of two
of block k at byte k, exponent + 127; the bytes past K/32 are 127).
"""

import math
import os
import sys

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def _mxfp4():
    path = os.path.join(os.getcwd(), "oko-xpu-kernels_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from xpu_kernels import mxfp4
    return mxfp4


def _moe():
    _mxfp4()
    from xpu_kernels import moe
    return moe


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # one token's hidden state quantized and read back: launches and latency
        dict(name="quantize_token", kind="quantize", m=1, k=4096, dtype="bf16"),
        # the hidden states of a long ragged prefill
        dict(name="quantize_prefill", kind="quantize", m=16381, k=5120, dtype="bf16"),
        # a float32 checkpoint's weight converted on load
        dict(name="quantize_weight_f32", kind="quantize", m=10240, k=1280, dtype="f32"),
        # a projection for one token: the 4-bit weight read once
        dict(name="linear_token", kind="linear", m=1, k=4096, n=4096, dtype="bf16", grad=False),
        # a few dozen sequences decoded together
        dict(name="linear_batch", kind="linear", m=48, k=4096, n=14336, dtype="f16", grad=False),
        # the benchmark's headline projection
        dict(name="linear_up", kind="linear", m=4096, k=1280, n=10240, dtype="bf16", grad=False),
        # a wide model's projection over a long prefill
        dict(name="linear_large", kind="linear", m=8192, k=8192, n=8192, dtype="bf16", grad=False),
        # fine-tuning around a frozen 4-bit weight: forward, dx, bias gradient
        dict(name="linear_train", kind="linear", m=4096, k=1280, n=5120, dtype="bf16", grad=True),
        # routing of a few decoded tokens: sort, gather, weighted sum
        dict(name="route_decode", kind="route", t=4, top=8, experts=64, d=2048, dtype="bf16",
             dropped=False, grad=False),
        # a training batch's routing with its gradients, some slots over capacity
        dict(name="route_train", kind="route", t=8190, top=8, experts=64, d=2048, dtype="bf16",
             dropped=True, grad=True),
        # the up-projections of the experts that a few decoded tokens chose
        dict(name="experts_decode", kind="experts", t=4, top=4, experts=32, k=2048, n=2816,
             dtype="bf16", dropped=False, grad=False),
        # the experts' products of a training batch, forward and dx
        dict(name="experts_train", kind="experts", t=4095, top=4, experts=32, k=2048, n=2816,
             dtype="bf16", dropped=True, grad=True),
    ]


def _log_int(rng, lo, hi, step=1):
    """A multiple of ``step`` in [lo, hi], uniform in its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "route", "experts", "experts"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "quantize":
        return dict(kind=kind, m=_log_int(rng, 1, 16384), k=_log_int(rng, 256, 8192, 32),
                    dtype=dtype)
    if kind == "linear":
        grad = rng.random() < 0.35
        return dict(kind=kind, m=_log_int(rng, 64 if grad else 1, 8192),
                    k=_log_int(rng, 512, 8192, 32), n=_log_int(rng, 512, 8192, 8),
                    dtype="bf16" if grad else dtype, grad=grad)
    grad = rng.random() < 0.5
    experts = rng.choice([8, 16, 32, 60, 64])
    case = dict(kind=kind, t=_log_int(rng, 64 if grad else 1, 8192 if kind == "route" else 4096),
                top=rng.choice([1, 2, 4, 6, 8]) if kind == "route" else rng.choice([1, 2, 4]),
                experts=experts)
    if kind == "route":
        case.update(d=_log_int(rng, 512, 4096, 8))
    else:
        case.update(k=_log_int(rng, 512, 4096, 32), n=_log_int(rng, 512, 2816, 16))
    case.update(dtype="bf16" if kind == "experts" else dtype, dropped=rng.random() < 0.4,
                grad=grad)
    return case


# ------------------------------------------------------- MXFP4 in its plain form
def _scale_width(k):
    return -(-k // 512) * 16


def _pow2(n):
    """2^n of an int32 tensor, -126 <= n <= 127, in 32 bits."""
    return ((n + 127) << 23).view(torch.float32)


def _quant(x):
    """x [.., K] -> (values [.., K/32, 32] on the 4-bit grid with their sign, exponents
    [.., K/32] as int32, 128 for a block with an infinity or NaN), in 32 bits."""
    b = x.float().unflatten(-1, (-1, 32))
    a = b.abs()
    amax = a.amax(dim=-1)
    bits = amax.view(torch.int32)
    # floor(log2) from the exponent field; a subnormal maximum is below 2^-126, and
    # its exponent clamps to -127
    e = ((bits >> 23) - 127 - 2).clamp(min=-127)
    bad = ~torch.isfinite(b).all(dim=-1)
    e = torch.where(bad, 128, e)
    # x / 2^e by two exact factors, each a normal power of two
    half = torch.div(e, 2, rounding_mode="floor")
    v = (a * _pow2(-half)[..., None]) * _pow2(half - e)[..., None]
    q = ((v > 0.25) * 0.5 + (v >= 0.75) * 0.5 + (v > 1.25) * 0.5 + (v >= 1.75) * 0.5
         + (v > 2.5) * 1.0 + (v >= 3.5) * 1.0 + (v > 5.0) * 2.0)
    return torch.copysign(q, b), e


def _values(q, e):
    """What the codes stand for, [.., K] in 32 bits."""
    half = torch.div(e, 2, rounding_mode="floor")
    v = (q * _pow2(half)[..., None]) * _pow2(e - half)[..., None]
    return torch.where((e == 128)[..., None], float("nan"), v).flatten(-2)


def _pack(q, e, k):
    """(codes, scales) as a program holds them."""
    a = q.abs()
    c = ((a > 0.25) * 1 + (a > 0.75) * 1 + (a > 1.25) * 1 + (a > 1.75) * 1 + (a > 2.5) * 1
         + (a > 3.5) * 1 + (a > 5.0) * 1 + torch.signbit(q) * 8).to(torch.uint8).flatten(-2)
    codes = c[..., 0::2] | (c[..., 1::2] << 4)
    scales = torch.full((*e.shape[:-1], _scale_width(k)), 127, dtype=torch.uint8, device=q.device)
    scales[..., :e.shape[-1]] = (e + 127).to(torch.uint8)
    return codes.contiguous(), scales


def _unpack(codes, scales):
    """The weight's values [.., K] in 32 bits."""
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6],
                        device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    q = grid[c.int()].unflatten(-1, (-1, 32))
    return _values(q, scales[..., :q.shape[-2]].int() - 127)


# ------------------------------------------------------------------- the inputs
def _activation(gen, m, k, dtype):
    """A residual stream: N(0, 1), one channel in a hundred 30 times as large."""
    x = torch.randn(m, k, generator=gen, device=DEV)
    x[:, torch.randperm(k, generator=gen, device=DEV)[:max(1, k // 100)]] *= 30.0
    return x.to(TYPES[dtype])


def _ids(gen, t, top, experts, dropped):
    """A router's choices: distinct experts a token, some experts liked more than
    others; with ``dropped`` one slot in twenty is over its expert's capacity (-1)."""
    liking = torch.randn(experts, generator=gen, device=DEV) * 0.5
    score = torch.randn(t, experts, generator=gen, device=DEV) + liking
    p, ids = torch.softmax(score, -1).topk(top, dim=-1)
    if dropped:
        ids = torch.where(torch.rand(t, top, generator=gen, device=DEV) < 0.05, -1, ids)
    return ids.to(torch.int32), p / p.sum(-1, keepdim=True)


def _sorted(ids, experts):
    """(order [S], position [T, k], offsets [E + 1]), all int32."""
    flat = ids.reshape(-1)
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    key, order = torch.sort(key, stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=order.device)
    offsets = torch.searchsorted(key, torch.arange(experts + 1, device=key.device,
                                                   dtype=key.dtype))
    return order.int(), position.int().reshape(ids.shape), offsets.int()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, dtype = case["kind"], TYPES[case["dtype"]]
    if kind == "quantize":
        return dict(case, x=_activation(gen, case["m"], case["k"], case["dtype"]))
    if kind == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        s = dict(case, x=_activation(gen, m, k, case["dtype"]))
        w = torch.randn(n, k, generator=gen, device=DEV) * 0.02
        s["codes"], s["scales"] = _pack(*_quant(w), k)
        s["bias"] = (torch.randn(n, generator=gen, device=DEV) * 0.01).to(dtype)
        if case["grad"]:
            s["x"].requires_grad_()
            s["bias"].requires_grad_()
            s["dy"] = torch.randn(m, n, generator=gen, device=DEV).to(dtype)
        return s
    t, top, experts = case["t"], case["top"], case["experts"]
    ids, weights = _ids(gen, t, top, experts, case["dropped"])
    if kind == "route":
        d = case["d"]
        s = dict(case, ids=ids, weights=weights, x=_activation(gen, t, d, case["dtype"]),
                 z=torch.randn(t * top, d, generator=gen, device=DEV).to(dtype))
        if case["grad"]:
            for name in ("weights", "x", "z"):
                s[name].requires_grad_()
            s["dxs"] = torch.randn(t * top, d, generator=gen, device=DEV).to(dtype)
            s["dy"] = torch.randn(t, d, generator=gen, device=DEV).to(dtype)
        return s
    k, n = case["k"], case["n"]
    s = dict(case, x=_activation(gen, t, k, case["dtype"]))
    w = torch.randn(experts, n, k, generator=gen, device=DEV) * 0.02
    s["codes"], s["scales"] = _pack(*_quant(w), k)
    s["order"], s["position"], s["offsets"] = _sorted(ids, experts)
    s["rows"] = torch.div(s["order"], top, rounding_mode="floor").int()
    # the plain form's padded batch: the most rows of one expert
    s["most"] = max(1, int((s["offsets"][1:] - s["offsets"][:-1]).max()))
    if case["grad"]:
        s["x"].requires_grad_()
        s["dy"] = torch.randn(t * top, n, generator=gen, device=DEV).to(dtype)
    return s


# --------------------------------------------------------------- the plain forms
def _plain_linear(s):
    x, dtype = s["x"].detach(), s["x"].dtype
    w = _unpack(s["codes"], s["scales"])
    out = {"y": (_values(*_quant(x)) @ w.t() + s["bias"].detach().float()).to(dtype)}
    if s["grad"]:
        dy = s["dy"].float()
        out["dx"] = (dy @ w).to(dtype)
        out["dbias"] = dy.sum(0).to(dtype)
    return out


def _plain_route(s):
    x, z, weights = s["x"].detach(), s["z"].detach(), s["weights"].detach()
    dtype, t, top = x.dtype, s["t"], s["top"]
    order, position, offsets = _sorted(s["ids"], s["experts"])
    live = torch.arange(t * top, device=x.device) < offsets[-1]
    token = order // top
    kept = (position < offsets[-1])[..., None]
    at = position.long()
    xs = torch.where(live[:, None], x[token], 0)
    zf = torch.where(kept, z[at].float(), 0)
    y = (weights[..., None] * zf).sum(1).to(dtype)
    out = dict(order=order, position=position, offsets=offsets, xs=xs, y=y)
    if s["grad"]:
        dy = s["dy"].float()
        out["dx"] = torch.where(kept, s["dxs"][at].float(), 0).sum(1).to(dtype)
        out["dz"] = torch.where(live[:, None], weights.reshape(-1)[order, None] * dy[token],
                                0).to(dtype)
        out["dweights"] = (zf * dy[:, None, :]).sum(-1)
    return out


def _plain_experts(s):
    x, rows, offsets, experts = s["x"].detach(), s["rows"], s["offsets"], s["experts"]
    dtype, n, k = x.dtype, s["n"], s["k"]
    i = torch.arange(rows.numel(), device=x.device, dtype=torch.int32)
    e = torch.searchsorted(offsets[1:], i, right=True)
    live = e < experts
    e = e.clamp(max=experts - 1)
    xs = _values(*_quant(x))[rows]
    if rows.numel() <= experts and not s["grad"]:          # a weight for each row
        w = _unpack(s["codes"][e], s["scales"][e])
        y = torch.bmm(w, xs[:, :, None])[:, :, 0]
        return {"y": torch.where(live[:, None], y, 0).to(dtype)}
    # the rows of each expert, padded to the most that one has
    w = _unpack(s["codes"], s["scales"])
    at = torch.where(live, e * s["most"] + (i - offsets[e]), experts * s["most"])
    size = experts * s["most"] + 1

    def product(rows_of, right):
        padded = rows_of.new_zeros(size, rows_of.shape[1])
        padded[at] = rows_of
        y = torch.bmm(padded[:-1].reshape(experts, s["most"], -1), right).flatten(0, 1)
        return torch.where(live[:, None], y[at.clamp(max=size - 2)], 0)

    out = {"y": product(xs, w.transpose(1, 2)).to(dtype)}
    if s["grad"]:
        dxs = product(s["dy"].float(), w)
        out["dx"] = dxs[s["position"].long()].sum(1).to(dtype)     # (0 where not live)
    return out


# -------------------------------------------------------------- the library's calls
def _own_linear(s):
    y = _mxfp4().linear(s["x"], s["codes"], s["scales"], s["bias"])
    if not s["grad"]:
        return {"y": y}
    dx, dbias = torch.autograd.grad(y, (s["x"], s["bias"]), s["dy"])
    return {"y": y, "dx": dx, "dbias": dbias}


def _own_route(s):
    moe = _moe()
    routing = moe.sort(s["ids"], s["experts"])
    xs = moe.dispatch(s["x"], routing)
    y = moe.combine(s["z"], routing, s["weights"])
    out = dict(order=routing.order, position=routing.position, offsets=routing.offsets, xs=xs,
               y=y)
    if s["grad"]:
        out["dx"], out["dz"], out["dweights"] = torch.autograd.grad(
            (xs, y), (s["x"], s["z"], s["weights"]), (s["dxs"], s["dy"]))
    return out


def _own_experts(s):
    routing = _moe().Routing(s["order"], s["position"], s["rows"], s["offsets"])
    y = _mxfp4().grouped_linear(s["x"], s["codes"], s["scales"], routing, gather=True)
    if not s["grad"]:
        return {"y": y}
    dx, = torch.autograd.grad(y, (s["x"],), s["dy"])
    return {"y": y, "dx": dx}


def run(s):
    kind = s["kind"]
    if kind == "quantize":
        if own:
            mxfp4 = _mxfp4()
            return mxfp4.dequantize(*mxfp4.quantize(s["x"]), dtype=s["x"].dtype)
        return _values(*_quant(s["x"])).to(s["x"].dtype)
    if own:
        return {"linear": _own_linear, "route": _own_route, "experts": _own_experts}[kind](s)
    return {"linear": _plain_linear, "route": _plain_route, "experts": _plain_experts}[kind](s)


# -------------------------------------------------------------------- the floors
def work(case):
    kind, b = case["kind"], SIZE[case["dtype"]]
    if kind == "quantize":
        v = case["m"] * case["k"]
        # x read, the codes and scales written and read, the values written
        return {"bytes": v * (2 * b + 2 * (0.5 + 1 / 32)), "flops": 4.0 * v}
    if kind == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        w = n * k * (0.5 + 1 / 32)
        bytes_ = m * k * b + w + n * b + m * n * b
        if case["grad"]:
            bytes_ += m * n * b + w + m * k * b + n * b
        return {"bytes": bytes_, "flops": 2.0 * m * n * k * (2 if case["grad"] else 1)}
    t, s = case["t"], case["t"] * case["top"]
    if kind == "route":
        d = case["d"]
        # ids and weights, order, position and offsets, x and the rows, z and y
        bytes_ = s * 16 + case["experts"] * 4 + 2 * (s + t) * d * b
        flops = 2.0 * s * d
        if case["grad"]:
            # dxs and dx; dy, z again and dz, dweights
            bytes_ += (s + t) * d * b + (2 * s + t) * d * b + 8 * s
            flops *= 3.5
        return {"bytes": bytes_, "flops": flops}
    k, n, e = case["k"], case["n"], case["experts"]
    used = min(e, s)                       # the experts that can have rows
    w = used * n * k * (0.5 + 1 / 32)
    bytes_ = t * k * b + w + s * n * b + s * 4
    if case["grad"]:
        bytes_ += s * n * b + w + t * k * b
    return {"bytes": bytes_, "flops": 2.0 * s * n * k * (2 if case["grad"] else 1)}


# --------------------------------------------------------------- in 64 bits, apart
def _two(e):
    """2^e in 64 bits from an integer tensor."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _q64(x):
    """What MXFP4 makes of x [.., K], in 64 bits: a grid of step 2^(e + j) by the
    binade of each value, rounded to even, at most 6 x 2^e."""
    b = x.double().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    e = (torch.frexp(amax)[1] - 3).clamp(-127, 127)    # amax in [2^(e+2), 2^(e+3))
    s = _two(torch.where(amax == 0, -127, e))
    v = b / s
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
    q = (torch.round(v / step) * step).clamp(-6, 6) * s
    return torch.where(torch.isfinite(amax), q, float("nan")).flatten(-2)


def _w64(codes, scales):
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).double()
    sign = torch.where(c >= 8, -1.0, 1.0)
    m = c % 8
    v = torch.where(m < 4, m / 2, torch.where(m < 6, m - 2, 2 * m - 8))
    k = v.shape[-1]
    s = _two(scales[..., :k // 32].long() - 127)
    return sign * v * s.repeat_interleave(32, dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    x = s["x"].detach()
    if kind == "quantize":
        return _q64(x)
    if kind == "linear":
        w = _w64(s["codes"], s["scales"])
        out = {"y": _q64(x) @ w.t() + s["bias"].detach().double()}
        if case["grad"]:
            out["dx"] = s["dy"].double() @ w
            out["dbias"] = s["dy"].double().sum(0)
        return out
    t, top, experts = case["t"], case["top"], case["experts"]
    if kind == "route":
        ids, weights = s["ids"].cpu(), s["weights"].detach().double()
        z = s["z"].detach().double()
        y = torch.zeros(t, case["d"], dtype=torch.float64, device=DEV)
        dx, dz = torch.zeros_like(y), torch.zeros_like(z)
        xs = torch.zeros(t * top, case["d"], dtype=torch.float64, device=DEV)
        dw = torch.zeros_like(weights)
        at = 0
        flat = ids.reshape(-1)
        for e in range(experts):
            slots = torch.nonzero(flat == e)[:, 0].to(DEV)
            n = slots.numel()
            tok = slots // top
            w = weights.reshape(-1)[slots]
            xs[at:at + n] = x[tok].double()
            y.index_add_(0, tok, w[:, None] * z[at:at + n])
            if case["grad"]:
                dy = s["dy"].double()[tok]
                dx.index_add_(0, tok, s["dxs"][at:at + n].double())
                dz[at:at + n] = w[:, None] * dy
                dw.view(-1)[slots] = (dy * z[at:at + n]).sum(-1)
            at += n
        out = dict(order=None, position=None, offsets=None, xs=xs, y=y)
        if case["grad"]:
            out.update(dx=dx, dz=dz, dweights=dw)
        return out
    off = s["offsets"].tolist()
    rows = s["rows"].long()
    xq = _q64(x)
    y = torch.zeros(t * top, case["n"], dtype=torch.float64, device=DEV)
    dx = torch.zeros(t, case["k"], dtype=torch.float64, device=DEV)
    for e in range(experts):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        w = _w64(s["codes"][e], s["scales"][e])
        y[a:b] = xq[rows[a:b]] @ w.t()
        if case["grad"]:
            dx.index_add_(0, rows[a:b], s["dy"][a:b].double() @ w)
    return {"y": y, "dx": dx} if case["grad"] else {"y": y}
