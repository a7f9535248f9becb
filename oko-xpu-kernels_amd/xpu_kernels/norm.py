"""RMS norm on gfx950: with the residual's addition, its gradients, and with an int8
output for the int8 linears.

    y = norm.rms_norm(x, weight)                          # [.., K] in x's type
    y, h = norm.rms_norm(x, weight, residual=r)           # h = x + r, y the norm of h
    q, scale, h = norm.rms_norm_int8(x, weight, residual=r)
    out = int8.linear_quantized(q, scale, w8, w_scale)    # of prepare_weight's w8 (many rows:
                                                          # see there)

``y = h / sqrt(mean(h^2) + eps) * weight`` over the last dimension, in fp32 from the
values of ``h`` in its type (bf16, fp16 or fp32) to the one rounding of ``y``; a sum of
squares beyond fp32's range makes the row zeros, as in fp32 arithmetic.  ``weight`` [K]
is of any of the three types, or None for ones.  All of it runs in ``libxpuint8.so`` on
torch's current stream without synchronising; there is no counterpart in the reference.
Rows may lie evenly apart, or in even runs as the heads in the columns of a projection do
(``qkv[..., :H * D].unflatten(-1, (H, D))``); other layouts are copied first.
"""

from __future__ import annotations

import torch

from .int8 import _lib as L
from .mxfp4 import TYPES, _check_float, _check_leaves, _opt, _wants_grad, _work

__all__ = ["rms_norm", "rms_norm_int8"]

GROUP = 256


def _check(x, weight, eps, residual):
    _check_float(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [.., K] with K >= 1, got {tuple(x.shape)}")
    if not isinstance(eps, (int, float)) or not eps >= 0:
        raise ValueError(f"eps must be a number >= 0, got {eps!r}")
    if weight is not None:
        _check_float(weight, "weight")
        if weight.shape != (x.shape[-1],):
            raise ValueError(f"weight must have shape ({x.shape[-1]},), got {tuple(weight.shape)}")
        if weight.device != x.device:
            raise TypeError(f"weight is on {weight.device} but x is on {x.device}")
    if residual is not None:
        if not isinstance(residual, torch.Tensor) or residual.dtype != x.dtype:
            raise TypeError(f"residual must be a {x.dtype} tensor as x is, got "
                            f"{getattr(residual, 'dtype', type(residual).__name__)}")
        if residual.shape != x.shape:
            raise ValueError(f"residual must have x's shape {tuple(x.shape)}, got "
                             f"{tuple(residual.shape)}")
        if residual.device != x.device:
            raise TypeError(f"residual is on {residual.device} but x is on {x.device}")


def _runs(x):
    """(inner, ld, outer) of the rows of ``x`` [.., K]: runs of ``inner`` rows, ld apart, runs
    outer apart; None for rows that do not lie so, or overlap."""
    k = x.shape[-1]
    if x.stride(-1) != 1 and k > 1:
        return None
    levels = []                                  # (rows, stride), the innermost first
    for n, s in reversed(list(zip(x.shape[:-1], x.stride()[:-1]))):
        if n == 1:
            continue
        if levels and s == levels[-1][0] * levels[-1][1]:
            levels[-1] = (levels[-1][0] * n, levels[-1][1])
        else:
            levels.append((n, s))
    if not levels:
        return 1, k, k
    if len(levels) > 2 or levels[0][1] < k:
        return None
    if len(levels) == 1:
        return 1, levels[0][1], levels[0][1]
    return levels[0][0], levels[0][1], levels[1][1]


def _lines(*tensors):
    """The inputs (some None) as the kernels read them: (inner, [(tensor, ld, outer)])."""
    tensors = [None if t is None else t.resolve_neg() for t in tensors]
    runs = [None if t is None else _runs(t) for t in tensors]
    inner = next((r[0] for r in runs if r is not None and r[0] > 1), 1)
    out = []
    for t, r in zip(tensors, runs):
        if t is None:
            out.append((None, 0, 0))
            continue
        if r is None or r[0] not in (1, inner):
            t = t.contiguous()
            r = 1, t.shape[-1], t.shape[-1]
        if r[0] != inner:
            r = inner, r[2], r[2] * inner
        out.append((t, r[1], r[2]))
    return inner, out


def _weight(weight):
    """(the weight dense, its type's number)"""
    if weight is None:
        return None, 0
    return weight.resolve_neg().contiguous(), TYPES[weight.dtype]


def _forward(x, weight, eps, residual):
    """(y, h): h is None without a residual."""
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = None if residual is None else torch.empty_like(y)
    if x.numel():
        inner, ((x2, ldx, ox), (r2, ldr, outer_r)) = _lines(x, residual)
        w, wt = _weight(weight)
        k = x.shape[-1]
        lib = L._lib()
        with L._on(x.device):
            if lib.xpuint8_rms_norm_stream(L._stream(x.device), x2.data_ptr(), TYPES[x.dtype], ldx,
                                           ox, _opt(r2), ldr, outer_r, inner, _opt(w), wt, eps,
                                           _opt(h), y.data_ptr(), x.numel() // k, k) != 0:
                L._err(lib, "norm.rms_norm")
    return y, h


def _backward(dy, h, weight, dh, eps, want_dweight):
    """(dx in h's shape, dweight or None)"""
    dx = torch.empty(h.shape, dtype=h.dtype, device=h.device)
    dweight = torch.empty_like(weight, memory_format=torch.contiguous_format) if want_dweight else None
    if not h.numel():
        return dx, dweight.zero_() if want_dweight else None
    k = h.shape[-1]
    m = h.numel() // k
    inner, ((h2, ldh, oh), (dy2, ldy, oy), (dh2, lddh, odh)) = _lines(h, dy, dh)
    w, wt = _weight(weight)
    lib = L._lib()
    need = lib.xpuint8_rms_norm_grad_workspace_size(m, k) if want_dweight else 0
    work = _work(need, h2)
    with L._on(h.device):
        if lib.xpuint8_rms_norm_grad_stream(L._stream(h.device), dy2.data_ptr(), TYPES[h.dtype], ldy,
                                            oy, h2.data_ptr(), ldh, oh, _opt(w), wt, _opt(dh2),
                                            lddh, odh, inner, eps, dx.data_ptr(), _opt(dweight), m,
                                            k, _opt(work), need) != 0:
            L._err(lib, "norm.rms_norm (gradient)")
    return dx, dweight


class _NormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        ctx.set_materialize_grads(False)
        y, h = _forward(x, weight, eps, residual)
        ctx.eps = eps
        ctx.save_for_backward(x if h is None else h, weight)
        return y if h is None else (y, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        L.check_backward(dy, dh)
        h, weight = ctx.saved_tensors
        want = ctx.needs_input_grad[1]
        if dy is None:                       # only h went on
            dx, dweight = dh, torch.zeros_like(weight) if want else None
        else:
            dx, dweight = _backward(dy, h, weight, dh, ctx.eps, want)
        return (dx if ctx.needs_input_grad[0] else None, dweight, None,
                dx if ctx.needs_input_grad[3] else None)


def rms_norm(x, weight=None, eps=1e-6, residual=None):
    """The RMS norm of ``x`` [.., K] times ``weight`` [K]; with ``residual`` (x's shape and
    type) of ``h = x + residual``, rounded to the type, and then ``(y, h)``.  Gradients
    reach x, weight and residual, through y and h; the weight's is summed in fp32 in a
    fixed order and rounded once."""
    if L.HOST is not None:
        r = L.HOST.rms_norm(x, weight, eps, residual)
        if r is not None:
            return r
    _check(x, weight, eps, residual)
    eps = float(eps)
    if _wants_grad(x, weight, residual):
        _check_leaves(x, weight, residual)
        return _NormFn.apply(x, weight, eps, residual)
    y, h = _forward(x, weight, eps, residual)
    return y if h is None else (y, h)


def rms_norm_int8(x, weight=None, eps=1e-6, residual=None, rotate=True):
    """:func:`rms_norm` with an int8 output: ``(q int8 [.., K], scale fp32 [..])``, and with
    ``residual`` ``h`` third; ``q * scale`` is the norm, with ``rotate`` rotated as
    :func:`int8.quantize` rotates (K a multiple of 256), for a weight of
    :func:`int8.prepare_weight`; without, for one quantized as it is
    (:func:`int8.quantize_row`).

    ``v = h * weight`` (rotated) in fp32, ``m = max(|v|, 1e-30)``,
    ``q = rint(v * (127 / m))`` and ``scale = m / 127 / sqrt(mean(h^2) + eps)``: the norm
    is not rounded between, and a row with an infinity or NaN has a NaN scale (as every row
    has with a NaN in the weight; finite rows whose squares overflow have a scale of 0, or
    NaN where ``v`` overflows too).
    Whole numbers have no gradient: inputs that need one are refused outside of
    ``torch.no_grad()``."""
    if L.HOST is not None:
        r = L.HOST.rms_norm_int8(x, weight, eps, residual, rotate)
        if r is not None:
            return r
    _check(x, weight, eps, residual)
    k = x.shape[-1]
    if rotate and k % GROUP:
        raise ValueError(f"K={k} is not a multiple of the ConvRot group size ({GROUP}); "
                         f"rotate=False takes any")
    if _wants_grad(x, weight, residual):
        raise RuntimeError("rms_norm_int8 has no gradient; call it under torch.no_grad(), or "
                           "rms_norm for one")
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    h = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x.numel():
        inner, ((x2, ldx, ox), (r2, ldr, outer_r)) = _lines(x, residual)
        w, wt = _weight(weight)
        lib = L._lib()
        with L._on(x.device):
            if lib.xpuint8_rms_norm_int8_stream(L._stream(x.device), x2.data_ptr(), TYPES[x.dtype],
                                                ldx, ox, _opt(r2), ldr, outer_r, inner, _opt(w), wt,
                                                float(eps), _opt(h), q.data_ptr(), scale.data_ptr(),
                                                1 if rotate else 0, x.numel() // k, k) != 0:
                L._err(lib, "norm.rms_norm_int8")
    return (q, scale) if h is None else (q, scale, h)
