"""The operators between a block's projections in 64 bits, on the CPU: RMS norm and its
gradient, its int8 form, the choice of experts and its gradient, rotary positions on
several axes."""

import math

import torch


# ------------------------------------------------------------------------ RMS norm
def stream(x, residual):
    """h: the sum rounded to the type (one rounding of the exact sum)."""
    return x if residual is None else (x.double() + residual.double()).to(x.dtype)


def rms_norm(x, weight, eps, residual=None):
    """(y in 64 bits, h in the type, 1 / rms in 64 bits)."""
    h = stream(x, residual)
    r = (h.double().square().mean(-1, keepdim=True) + eps).rsqrt()
    w = 1.0 if weight is None else weight.double()
    return h.double() * r * w, h, r


def rms_norm_grad(dy, h, weight, eps, dh=None):
    """(dx, dweight) in 64 bits."""
    h, dy = h.double(), dy.double()
    r = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    g = dy if weight is None else dy * weight.double()
    dx = r * g - h * r ** 3 * (g * h).mean(-1, keepdim=True)
    return dx if dh is None else dx + dh.double(), (dy * h * r).flatten(0, -2).sum(0)


def rotation():
    """The 256-point rotation [256, 256]."""
    four = torch.tensor([[1, 1, 1, -1], [1, 1, -1, 1], [1, -1, 1, 1], [-1, 1, 1, 1]]).double() / 2
    two = torch.kron(four, four)
    return torch.kron(two, two)


def rms_norm_int8(x, weight, eps, residual=None, rotate=True):
    """(the unrounded codes, scales, h): codes lie where q is to be rounded from."""
    _, h, r = rms_norm(x, weight, eps, residual)
    v = h.double() * (1.0 if weight is None else weight.double())
    if rotate:
        v = (v.unflatten(-1, (-1, 256)) @ rotation().t()).flatten(-2)
    m = v.abs().amax(-1, keepdim=True).clamp(min=1e-30)
    return v * (127.0 / m), (m / 127.0 * r)[..., 0], h


# ------------------------------------------------------------- the choice of experts
LOWEST = -1e300       # a NaN key; a group of two has a finite value


def route(logits, top, scores="softmax", bias=None, groups=1, top_groups=1, renormalize=True,
          scale=1.0):
    """(ids, weights in 64 bits), a token at a time."""
    t, e = logits.shape
    n = e // groups
    ids = torch.full((t, top), -1, dtype=torch.int32)
    weights = torch.zeros(t, top, dtype=torch.float64)
    for i, row in enumerate(logits.double().tolist()):
        spoilt = any(math.isnan(v) or (scores == "softmax" and v == math.inf) for v in row)
        live = [j for j in range(e) if row[j] != -math.inf]
        if spoilt:
            key = {j: LOWEST if math.isnan(row[j]) else row[j] for j in live}
            s = {j: math.nan for j in live}
        elif scores == "softmax":
            most = max((row[j] for j in live), default=0.0)
            total = math.fsum(math.exp(row[j] - most) for j in live)
            s = {j: math.exp(row[j] - most) / total for j in live}
        else:
            s = {j: 1 / (1 + math.exp(-row[j])) if row[j] > -700 else math.exp(row[j]) for j in live}
        if not spoilt:
            b = [0.0] * e if bias is None else bias.double().tolist()
            # without a bias scores rise with their logits
            key = {j: row[j] if bias is None and groups == 1 else s[j] + b[j] for j in live}
        key = {j: LOWEST if math.isnan(v) else v for j, v in key.items() if v != -math.inf}
        if groups > 1:
            best = [sorted((key[j] for j in range(g * n, (g + 1) * n) if j in key), reverse=True)[:2]
                    for g in range(groups)]
            value = [sum(v) if v else -math.inf for v in best]
            kept = sorted(range(groups), key=lambda g: (-value[g], g))[:top_groups]
            key = {j: v for j, v in key.items() if j // n in kept}
        chosen = sorted(key, key=lambda j: (-key[j], j))[:top]
        ids[i, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
        if spoilt:
            weights[i] = math.nan
            continue
        if renormalize and chosen:
            # a common factor of the scores drops out
            if scores == "softmax":
                ref = max(row[j] for j in chosen)
                w = [math.exp(row[j] - ref) for j in chosen]
            else:
                ref = min(0.0, max(row[j] for j in chosen))
                w = [math.exp(row[j] - ref) / (1 + math.exp(row[j])) if row[j] < 0
                     else 1 / (1 + math.exp(-row[j])) for j in chosen]
            w = [v / math.fsum(w) for v in w]
        else:
            w = [s[j] for j in chosen]
        weights[i, :len(w)] = scale * torch.tensor(w, dtype=torch.float64)
    return ids, weights


def route_grad(logits, ids, dweights, scores="softmax", renormalize=True, scale=1.0):
    """dlogits in 64 bits of the weights' gradient, the choice held fixed: by torch's
    differentiation of the weights' formula.  NaNs for a token whose weights are."""
    lg = logits.double().clone().requires_grad_()
    live = ids >= 0
    at = ids.clamp(min=0).long()
    # log-scores: the softmax's, or -log(1 + e^-l)
    log_s = (torch.log_softmax(lg, -1) if scores == "softmax"
             else torch.nn.functional.logsigmoid(lg)).gather(1, at)
    log_s = log_s.masked_fill(~live, -math.inf)
    w = torch.softmax(log_s, -1) if renormalize else torch.exp(log_s)
    g = torch.where(live, dweights.double(), 0.0) * scale
    out = torch.zeros_like(lg)
    some = live.any(-1)
    if some.any():
        d, = torch.autograd.grad((torch.where(live, w, 0.0) * g)[some].sum(), lg)
        out[some] = d[some]
    spoilt = logits.isnan() if scores == "sigmoid" else logits.isnan() | (logits == math.inf)
    out[spoilt.any(-1)] = math.nan
    return out


# -------------------------------------------------------------------- rotary positions
def rotate_axes(x, positions, inv_freq, axis, split_half=True, inverse=False):
    """x [B, S, H, D] turned, in 64 bits; positions [A, B, S] or [A, S]."""
    b, s, _, d = x.shape
    p = positions.double()
    if p.dim() == 2:
        p = p[:, None].expand(-1, b, -1)
    n = inv_freq.numel()
    turned = torch.stack([p[a] if 0 <= a < p.shape[0] else torch.zeros(b, s).double()
                          for a in axis.tolist()], -1)
    angle = (turned * inv_freq.double() * (-1 if inverse else 1))[:, :, None]
    c, si = torch.cos(angle), torch.sin(angle)
    y = x.double().clone()
    first = slice(0, n) if split_half else slice(0, 2 * n, 2)
    second = slice(n, 2 * n) if split_half else slice(1, 2 * n, 2)
    u, v = y[..., first].clone(), y[..., second].clone()
    y[..., first] = u * c - v * si
    y[..., second] = v * c + u * si
    return y
