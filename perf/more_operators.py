"""Performance cases of what a transformer block does around its projections: RMS norm
with the residual's addition and its gradient, the same with an int8 output, routing
to experts with its gradient, and rotary positions on several axes with theirs.

``listed()`` are fixed cases, ``draw()`` gives more of the same ranges,
``prepare()`` makes what a program holds before the call and ``run()`` is one
pass: the plain form in elementary torch operations, or with ``own`` the library's
calls.  ``exact()`` restates each operator in 64 bits.
"""

import math
import os
import sys

import torch

own = False
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6


def _package(name):
    path = os.path.join(os.getcwd(), "oko-xpu-kernels_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    if name == "norm":
        from xpu_kernels import norm as module
    elif name == "moe":
        from xpu_kernels import moe as module
    else:
        from xpu_kernels import rope as module
    return module


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # one decoded token between two layers: launches and latency
        dict(name="norm_token", kind="norm", m=1, k=4096, dtype="bf16", residual=True, grad=False),
        # the residual stream of a long ragged prefill
        dict(name="norm_prefill", kind="norm", m=16381, k=5120, dtype="bf16", residual=True,
             grad=False),
        # the heads of a query normalised each by itself, forward and backward
        dict(name="norm_heads", kind="norm", m=4096 * 20, k=64, dtype="f16", residual=False,
             grad=True),
        # a training batch's norm with the gradient of both branches and of the weight
        dict(name="norm_train", kind="norm", m=8192, k=4096, dtype="bf16", residual=True, grad=True),
        # a few decoded sequences on their way into an int8 projection
        dict(name="int8_batch", kind="int8", m=16, k=4096, dtype="bf16", residual=True, rotate=True),
        # the activations of a prefill for the same
        dict(name="int8_prefill", kind="int8", m=16381, k=5120, dtype="bf16", residual=True,
             rotate=True),
        # without the rotation, for a weight quantized as it is; a float32 stream
        dict(name="int8_plain", kind="int8", m=4096, k=1280, dtype="f32", residual=True, rotate=False),
        # a few decoded tokens choose their experts
        dict(name="route_decode", kind="route", t=4, experts=64, top=8, dtype="bf16",
             scores="softmax", bias=False, groups=1, top_groups=1, renormalize=True, masked=False,
             grad=False),
        # a training batch's choice among groups, balanced by a bias
        dict(name="route_train", kind="route", t=16381, experts=256, top=8, dtype="f32",
             scores="sigmoid", bias=True, groups=8, top_groups=4, renormalize=True, masked=False,
             grad=True),
        # the queries and keys of a batch of decoded tokens
        dict(name="rope_decode", kind="rope", b=32, s=1, hq=32, hk=8, d=128, sections="16,24,24",
             shared=True, split=True, dtype="bf16", grad=False),
        # a video's tokens, each axis with frequencies of its own
        dict(name="rope_video", kind="rope", b=1, s=32760, hq=24, hk=24, d=128, sections="16,24,24",
             shared=False, split=False, dtype="bf16", grad=False),
        # images and text in training, some of the head left unrotated
        dict(name="rope_train", kind="rope", b=3, s=2047, hq=16, hk=4, d=80, sections="8,12,12",
             shared=True, split=True, dtype="f16", grad=True),
    ]


def _log_int(rng, lo, hi, step=1):
    """A multiple of ``step`` in [lo, hi], uniform in its logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["norm", "norm", "int8", "route", "route", "rope", "rope"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("norm", "int8"):
        rotate = rng.random() < 0.6
        step = 256 if kind == "int8" and rotate else rng.choice([1, 8, 8, 64])
        k = _log_int(rng, 256 if step == 256 else 64, 8192, step)
        case = dict(kind=kind, k=k, m=_log_int(rng, 1, min(65536, (1 << 25) // k)), dtype=dtype,
                    residual=rng.random() < 0.6)
        return dict(case, rotate=rotate) if kind == "int8" else dict(case, grad=rng.random() < 0.5)
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log_int(rng, 8, 512 // groups)
        top_groups = rng.randint(1, groups)
        return dict(kind=kind, t=_log_int(rng, 1, 16384), experts=experts,
                    top=rng.randint(1, min(8, top_groups * (experts // groups) // 4)), dtype=dtype,
                    scores=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5,
                    groups=groups, top_groups=top_groups, renormalize=rng.random() < 0.7,
                    masked=rng.random() < 0.2, grad=rng.random() < 0.5)
    axes = rng.choice([1, 2, 3, 3])
    sections = [rng.choice([4, 8, 8, 12, 16, 5]) for _ in range(axes)]
    hk = rng.choice([1, 2, 4, 8])
    s = _log_int(rng, 1, 16384)
    return dict(kind=kind, b=rng.randint(1, max(1, min(8, 16384 // s))), s=s,
                hq=hk * rng.choice([1, 2, 4]), hk=hk, d=2 * sum(sections) + rng.choice([0, 0, 16, 6]),
                sections=",".join(map(str, sections)), shared=rng.random() < 0.5,
                split=rng.random() < 0.6, dtype=dtype, grad=rng.random() < 0.4)


# ------------------------------------------------------------------- the inputs
def _activation(gen, m, k, dtype):
    """A residual stream: N(0, 1), one channel in a hundred 30 times as large."""
    x = torch.randn(m, k, generator=gen, device=DEV)
    x[:, torch.randperm(k, generator=gen, device=DEV)[:max(1, k // 100)]] *= 30.0
    return x.to(TYPES[dtype])


def _frequencies(sections, shared):
    """(inverse frequencies fp64 [P], the axis of each int32 [P]) of base 10000."""
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections))
    if shared:                      # one run of frequencies over all axes
        j, n = torch.arange(sum(sections)).double(), torch.tensor(float(sum(sections)))
    else:                           # each axis its own
        j = torch.cat([torch.arange(n) for n in sections]).double()
        n = torch.tensor(sections).repeat_interleave(torch.tensor(sections)).double()
    return (10000.0 ** (-j / n)).to(DEV), axis.int().to(DEV)


def _positions(gen, axes, b, s):
    """[axes, B, S] int32: a grid of frames, rows and columns behind a text of its own length."""
    i = torch.arange(s, device=DEV)
    width = max(1, int(math.sqrt(s) * 0.7))
    grid = [i // (width * width), i // width % width, i % width][-axes:]
    first = torch.randint(0, 30000, (b, 1), generator=gen, device=DEV)
    return torch.stack([g[None] + first for g in grid]).int()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, dtype = case["kind"], TYPES[case["dtype"]]
    s = dict(case)
    if kind in ("norm", "int8"):
        m, k = case["m"], case["k"]
        s["x"] = _activation(gen, m, k, case["dtype"])
        s["w"] = (1 + 0.1 * torch.randn(k, generator=gen, device=DEV)).to(dtype)
        s["r"] = (_activation(gen, m, k, case["dtype"]) if case["residual"] else None)
        if kind == "norm" and case["grad"]:
            s["dy"] = torch.randn(m, k, generator=gen, device=DEV).to(dtype)
            s["dh"] = (torch.randn(m, k, generator=gen, device=DEV).to(dtype)
                       if case["residual"] else None)
            for name in ("x", "w", "r"):
                if s[name] is not None:
                    s[name].requires_grad_()
        return s
    if kind == "route":
        t, experts = case["t"], case["experts"]
        liking = torch.randn(experts, generator=gen, device=DEV) * 0.5
        logits = torch.randn(t, experts, generator=gen, device=DEV) + liking
        if case["masked"]:            # experts that a token may not use
            logits[torch.rand(t, experts, generator=gen, device=DEV) < 0.1] = -math.inf
        s["logits"] = logits.to(dtype)
        s["offset"] = (torch.randn(experts, generator=gen, device=DEV) * 0.05
                       if case["bias"] else None)
        if case["grad"]:
            s["logits"].requires_grad_()
            s["dweights"] = torch.randn(t, case["top"], generator=gen, device=DEV)
        return s
    b, n, hq, hk, d = (case[name] for name in ("b", "s", "hq", "hk", "d"))
    sections = [int(v) for v in case["sections"].split(",")]
    s["inv_freq"], s["axis"] = _frequencies(sections, case["shared"])
    s["positions"] = _positions(gen, len(sections), b, n)
    # the columns of q and k in the output of one projection to q, k and v
    qkv = torch.randn(b, n, (hq + 2 * hk) * d, generator=gen, device=DEV).to(dtype)
    s["q"] = qkv[..., :hq * d].unflatten(-1, (hq, d))
    s["k"] = qkv[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
    if case["grad"]:
        for name in ("q", "k"):
            s["d" + name] = torch.randn(s[name].shape, generator=gen, device=DEV).to(dtype)
            s[name].requires_grad_()
    return s


# --------------------------------------------------------------- the plain forms
def _plain_stream(s):
    """The residual stream's new value in its own type, in 32 bits."""
    x = s["x"].detach()
    if s["r"] is not None:
        x = (x.float() + s["r"].detach().float()).to(x.dtype)
    return x.float()


def _plain_norm(s):
    dtype, w = s["x"].dtype, s["w"].detach().float()
    h = _plain_stream(s)
    r = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    n = h * r
    out = {"y": (n * w).to(dtype)}
    if s["r"] is not None:
        out["h"] = h.to(dtype)
    if s["grad"]:
        dy = s["dy"].float()
        g = dy * w
        dx = r * (g - n * (g * n).mean(-1, keepdim=True))
        if s["r"] is not None:
            dx = dx + s["dh"].float()
        out["dx"] = dx.to(dtype)
        if s["r"] is not None:
            out["dr"] = dx.to(dtype)
        out["dw"] = (dy * n).sum(0).to(dtype)
    return out


def _four(v, dim):
    """One axis of the rotation: 4 values to their sums with one sign turned each."""
    a, b, c, d = v.unbind(dim)
    p, q = a + b, a - b
    return torch.stack([(p + c) - d, (p - c) + d, (q + c) + d, (c - q) + d], dim)


def _four_pairs(v, dim):
    """The same sums in pairs (the order of the two outer axes)."""
    a, b, c, d = v.unbind(dim)
    p, q, r, t = a + b, a - b, c + d, c - d
    return torch.stack([p + t, p - t, q + r, r - q], dim)


def _rotated(v):
    """v [.., K] rotated by 256s, in 32 bits and the order that the codes are defined by:
    the last base-4 digit of an element's place first."""
    u = v.unflatten(-1, (-1, 4, 4, 4, 4))
    u = _four_pairs(_four_pairs(_four(_four(u, -1), -2), -3), -4)
    return u.flatten(-5) * 0.0625


def _plain_int8(s):
    h = _plain_stream(s)
    r = torch.rsqrt(h.square().mean(-1) + EPS)
    v = h * s["w"].float()
    if s["rotate"]:
        v = _rotated(v)
    m = v.abs().amax(-1).clamp(min=1e-30)
    # (a quotient that is the nearest 32-bit value: codes next to a border go by it)
    inv = (127.0 / m.double()).float()
    # the codes are whole numbers that stand for code * scale; both are returned
    out = {"q": torch.round(v * inv[:, None]).to(torch.int8), "scale": r * m / 127.0}
    if s["r"] is not None:
        out["h"] = h.to(s["x"].dtype)
    return out


def _first(values, n):
    """The places of the n largest along the last dimension, equal ones in order of place."""
    return torch.sort(values, dim=-1, descending=True, stable=True)[1][..., :n]


def _plain_route(s):
    # in 64 bits: which experts are chosen hangs on values next to each other
    logits = s["logits"].detach().double()
    if s["scores"] == "softmax":
        p = torch.exp(logits - logits.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-logits))
    key = p if s["offset"] is None else p + s["offset"].double()
    key = torch.where(logits == -math.inf, -math.inf, key)
    if s["groups"] > 1:
        by = key.unflatten(-1, (s["groups"], -1))
        two = torch.sort(by, dim=-1, descending=True)[0][..., :2]
        two[..., 1:] = torch.where(two[..., 1:] == -math.inf, 0.0, two[..., 1:])
        kept = torch.zeros_like(two[..., 0], dtype=torch.bool)
        kept.scatter_(1, _first(two.sum(-1), s["top_groups"]), True)
        key = torch.where(kept[..., None], by, -math.inf).flatten(-2)
    at = _first(key, s["top"])
    live = key.gather(1, at) > -math.inf
    chosen = torch.where(live, p.gather(1, at), 0.0)
    total = chosen.sum(-1, keepdim=True) if s["renormalize"] else 1.0
    weights = chosen / total
    out = {"ids": torch.where(live, at, -1).int(), "weights": weights.float()}
    if s["grad"]:
        g = torch.where(live, s["dweights"].double(), 0.0)
        # the gradient of the chosen scores, then of all logits
        if s["renormalize"]:
            g = (g - (g * weights).sum(-1, keepdim=True)) / total
        dp = torch.zeros_like(p).scatter_add_(1, at, g)
        if s["scores"] == "softmax":
            d = p * (dp - (p * dp).sum(-1, keepdim=True))
        else:
            d = dp * p * (1.0 - p)
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def _plain_rotate(x, cos, sin, split, back=False):
    """The first 2 P elements of each head rotated pair by pair, in 32 bits."""
    n = cos.shape[-1]
    f = x.float()
    turned = f[..., :2 * n].unflatten(-1, (2, n) if split else (n, 2))
    a, b = turned.unbind(-2 if split else -1)
    sin = -sin if back else sin
    turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -2 if split else -1)
    return torch.cat([turned.flatten(-2), f[..., 2 * n:]], -1).to(x.dtype)


def _plain_rope(s):
    # far positions lose their angle in 32 bits
    angle = s["positions"].double()[s["axis"].long()].movedim(0, -1) * s["inv_freq"]
    cos, sin = (f(angle).float()[:, :, None] for f in (torch.cos, torch.sin))
    out = {name: _plain_rotate(s[name].detach(), cos, sin, s["split"]) for name in ("q", "k")}
    if s["grad"]:
        for name in ("dq", "dk"):
            out[name] = _plain_rotate(s[name], cos, sin, s["split"], back=True)
    return out


# -------------------------------------------------------------- the library's calls
def _own_norm(s):
    y = _package("norm").rms_norm(s["x"], s["w"], EPS, residual=s["r"])
    if s["r"] is None:
        out, inputs, results, grads = {"y": y}, ("x", "w"), (y,), (s.get("dy"),)
    else:
        out, inputs = {"y": y[0], "h": y[1]}, ("x", "w", "r")
        results, grads = y, (s.get("dy"), s.get("dh"))
    if s["grad"]:
        got = torch.autograd.grad(results, [s[n] for n in inputs], grads)
        out.update(("d" + n, g) for n, g in zip(inputs, got))
    return out


def _own_int8(s):
    got = _package("norm").rms_norm_int8(s["x"], s["w"], EPS, residual=s["r"], rotate=s["rotate"])
    return dict(zip(("q", "scale", "h"), got))


def _own_route(s):
    ids, weights = _package("moe").route(
        s["logits"], s["top"], scores=s["scores"], bias=s["offset"], groups=s["groups"],
        top_groups=s["top_groups"], renormalize=s["renormalize"])
    out = {"ids": ids, "weights": weights}
    if s["grad"]:
        out["dlogits"], = torch.autograd.grad(weights, s["logits"], s["dweights"])
    return out


def _own_rope(s):
    rope = _package("rope")
    q, k = rope.rotate_axes(s["q"], s["k"], s["positions"],
                            rope.AxisFrequencies(s["inv_freq"], s["axis"]), split_half=s["split"])
    out = {"q": q, "k": k}
    if s["grad"]:
        out["dq"], out["dk"] = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    return out


def run(s):
    kind = s["kind"]
    if own:
        return {"norm": _own_norm, "int8": _own_int8, "route": _own_route, "rope": _own_rope}[kind](s)
    return {"norm": _plain_norm, "int8": _plain_int8, "route": _plain_route,
            "rope": _plain_rope}[kind](s)


# -------------------------------------------------------------------- the floors
def work(case):
    kind, b = case["kind"], SIZE[case["dtype"]]
    if kind in ("norm", "int8"):
        v, k = float(case["m"] * case["k"]), case["k"]
        bytes_ = v * b * (3 if case["residual"] else 1) + k * b        # x, residual, h; w
        if kind == "int8":
            return {"bytes": bytes_ + v + case["m"] * 4,
                    "flops": v * (6 + (12 if case["rotate"] else 0))}
        bytes_ += v * b
        if case["grad"]:      # dy, what was normalised, dx; dh; the weight and its gradient
            bytes_ += v * b * (4 if case["residual"] else 3) + 2 * k * b
        return {"bytes": bytes_, "flops": v * (15 if case["grad"] else 5)}
    if kind == "route":
        t, e, top = case["t"], case["experts"], case["top"]
        bytes_ = t * e * b + t * top * 8 + (e * 4 if case["bias"] else 0)
        if case["grad"]:      # dweights, the ids and the logits again, dlogits
            bytes_ += t * top * 8 + 2 * t * e * b
        return {"bytes": bytes_, "flops": t * e * (20.0 + top)}
    axes = case["sections"].count(",") + 1
    v = float(case["b"] * case["s"] * (case["hq"] + case["hk"]) * case["d"])
    passes = 2 if case["grad"] else 1
    return {"bytes": passes * (2 * v * b + 4.0 * axes * case["b"] * case["s"]),
            "flops": passes * 3 * v}


# --------------------------------------------------------------- in 64 bits, apart
def _exact_norm(s):
    h = s["x"].detach()
    if s["r"] is not None:       # the stream's new value is kept in its type
        h = (h.double() + s["r"].detach().double()).to(h.dtype)
    h, w = h.double(), s["w"].detach().double()
    rms = (h.pow(2).sum(-1, keepdim=True) / s["k"] + EPS).sqrt()
    if s["kind"] == "int8":
        v = h * w
        if s["rotate"]:
            one = torch.ones(4, 4, dtype=torch.float64) - 2 * torch.eye(4, dtype=torch.float64).flip(0)
            four = torch.kron(torch.kron(one, one), torch.kron(one, one)).to(DEV) / 16
            v = (v.reshape(-1, 256) @ four.t()).reshape(h.shape)
        scale = (v.abs().amax(-1).clamp(min=1e-30) / 127) / rms[:, 0]
        return {"q": None, "scale": scale, **({"h": h} if s["r"] is not None else {})}
    out = {"y": h / rms * w}
    if s["r"] is not None:
        out["h"] = h
    if s["grad"]:
        dy = s["dy"].double()
        along = (dy * w * h).sum(-1, keepdim=True) / (s["k"] * rms.pow(3))
        dx = dy * w / rms - h * along
        if s["r"] is not None:
            dx += s["dh"].double()
            out["dr"] = dx
        out["dx"] = dx
        out["dw"] = (dy * (h / rms)).sum(0)
    return out


def _exact_route(s):
    logits = s["logits"].detach().double()
    t, experts, top = s["t"], s["experts"], s["top"]
    soft = s["scores"] == "softmax"
    log_p = (logits - torch.logsumexp(logits, -1, keepdim=True) if soft
             else -torch.log1p(torch.exp(-logits)))
    p = torch.exp(log_p)
    key = p + (0.0 if s["offset"] is None else s["offset"].double())
    key[logits == -math.inf] = -math.inf
    n = experts // s["groups"]
    if s["groups"] > 1:
        value = torch.stack([key[:, g * n:(g + 1) * n].topk(min(2, n))[0].clamp(min=-9.0)
                             .where(key[:, g * n:(g + 1) * n].topk(min(2, n))[0] > -math.inf, 0.0)
                             .sum(-1) for g in range(s["groups"])], -1)
        order = torch.argsort(-value, dim=-1, stable=True)
        for j in range(s["top_groups"], s["groups"]):
            out_of = order[:, j:j + 1] * n + torch.arange(n, device=DEV)
            key.scatter_(1, out_of, -math.inf)
    order = torch.argsort(-key, dim=-1, stable=True)[:, :top]
    live = torch.isfinite(key.gather(1, order))
    log_w = log_p.gather(1, order).masked_fill(~live, -math.inf)
    if s["renormalize"]:
        log_w = log_w - torch.logsumexp(log_w, -1, keepdim=True)
    weights = torch.exp(log_w)
    out = {"ids": None, "weights": weights}
    if s["grad"]:
        g = s["dweights"].double().masked_fill(~live, 0.0)
        # through the logarithms of the weights, then of the scores
        d = g * weights
        if s["renormalize"]:
            d = d - weights * d.sum(-1, keepdim=True)
        full = torch.zeros(t, experts, dtype=torch.float64, device=DEV).scatter_add_(1, order, d)
        out["dlogits"] = (full - p * full.sum(-1, keepdim=True) if soft else full * (1 - p))
    return out


def _exact_rope(s):
    split, n = s["split"], s["inv_freq"].numel()
    z = torch.polar(torch.ones(1, dtype=torch.float64, device=DEV),
                    torch.stack([s["positions"][a].double() * f for a, f in
                                 zip(s["axis"].tolist(), s["inv_freq"].tolist())], -1))[:, :, None]
    first = torch.arange(n, device=DEV) if split else 2 * torch.arange(n, device=DEV)
    second = first + (n if split else 1)
    out = {}
    for name, turn in (("q", z), ("k", z), ("dq", z.conj()), ("dk", z.conj())):
        if name not in s:
            continue
        y = s[name].detach().double().clone()
        v = torch.complex(y[..., first], y[..., second]) * turn
        y[..., first], y[..., second] = v.real, v.imag
        out[name] = y
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "int8": _exact_norm, "route": _exact_route,
            "rope": _exact_rope}[case["kind"]](s)
