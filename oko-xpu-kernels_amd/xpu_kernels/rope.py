"""Rotary embeddings: of q/k read from the int8 GEMM's accumulator with their RMSNorm, and
of q/k by positions on several axes (:func:`rotate_axes`: text, images, video).

The fused consumer of a quantized qkv projection
(okolenmi/oko-xpu-kernels ``python/xpu_kernels/triton/rope.py:378-405, 643-652``,
``_rows_dq`` and ``rms_rope_split_half_dequant``): the int32 accumulator slice
of q (or k), [B, S, H, D], is dequantized with the epilogue's expression and
bf16 rounding, RMS-normalized per head row, scaled, and rotated pairwise by
``freqs_cis`` [FB, FS, 1, D/2, 2, 2] in one HIP kernel
(``xpuint8_rms_rope_dequant_stream``).  The reference runs a Triton kernel
behind a self-test gate; here the HIP kernel is the only path.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from .int8 import _lib as L
from .mxfp4 import TYPES, _check_float, _check_leaves, _opt, _wants_grad

__all__ = ["AxisFrequencies", "axis_frequencies", "rms_rope_split_half_dequant", "rotate_axes",
           "rows_dq"]

POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
MAX_PAIRS, MAX_HEAD_DIM, MAX_AXES, MAX_HEADS = 512, 4096, 16, 65536


def _f32(t, name):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype != torch.float32:
        t = t.to(torch.float32)
    return t


def rows_dq(acc, freqs_cis, scale, epsilon, x_scale, w_scale, split_half=True):
    """RMSNorm + rope of one [B, S, H, D] int32 accumulator slice -> bf16
    [B, S, H, D] (rope.py:378-405).

    ``acc``'s head dim must be contiguous (a column slice of a wider qkv
    accumulator is fine); ``x_scale`` is the quantizer's per-row scale, [B, S]
    (or [B*S]); ``w_scale`` the projection's per-column scale of this slice,
    [H*D]; ``scale`` the per-dim norm weight, [D]."""
    if not isinstance(acc, torch.Tensor) or acc.dtype != torch.int32 or acc.dim() != 4:
        raise TypeError("acc must be an int32 [B, S, H, D] tensor")
    if acc.device.type != "cuda":
        raise TypeError(f"expected a GPU (ROCm) tensor, got {acc.device}")
    B, S, H, D = acc.shape
    if acc.stride(3) != 1:
        raise ValueError("acc's head dimension must be contiguous")
    f = _f32(freqs_cis, "freqs_cis")
    if f.dim() != 6 or tuple(f.shape[3:]) != (D // 2, 2, 2) or f.shape[2] != 1:
        raise ValueError(f"freqs_cis must be [B or 1, S or 1, 1, {D // 2}, 2, 2], "
                         f"got {tuple(f.shape)}")
    if f.shape[0] not in (1, B) or f.shape[1] not in (1, S):
        raise ValueError(f"freqs_cis {tuple(f.shape)} does not broadcast over B={B}, S={S}")
    sc = _f32(scale, "scale").contiguous()
    if sc.numel() != D:
        raise ValueError(f"scale must have D={D} values")
    xs = _f32(x_scale, "x_scale")
    if xs.numel() != B * S:
        raise ValueError(f"x_scale must have B*S={B * S} values")
    xs = xs.reshape(B, S)
    ws = _f32(w_scale, "w_scale").contiguous()
    if ws.numel() != H * D:
        raise ValueError("w_scale must cover H * D columns")
    for t, name in ((f, "freqs_cis"), (sc, "scale"), (xs, "x_scale"), (ws, "w_scale")):
        if t.device != acc.device:
            raise TypeError(f"{name} is on {t.device} but acc is on {acc.device}")
    out = torch.empty((B, S, H, D), dtype=torch.bfloat16, device=acc.device)
    lib = L._lib()
    rc = lib.xpuint8_rms_rope_dequant_stream(
        L._stream(acc.device), L._ptr(acc), acc.stride(0), acc.stride(1), acc.stride(2),
        L._ptr(xs), xs.stride(0), xs.stride(1), L._ptr(ws), L._ptr(f),
        f.stride(0), f.stride(1), f.stride(3), f.stride(4), f.stride(5), f.shape[0], f.shape[1],
        L._ptr(sc), L._ptr(out), B, S, H, D, float(epsilon), 1 if split_half else 0)
    if rc != 0:
        L._err(lib, "rms_rope_dequant")
    return out


def rms_rope_split_half_dequant(q_acc, k_acc, freqs_cis, q_w, k_w, x_scale, q_scale,
                                k_scale=None, epsilon=1e-6, split_half=True):
    """``rms_rope_split_half`` with the INT8 dequant folded into the load
    (rope.py:643-652): returns (q, k) bf16 [B, S, H, D]."""
    if k_scale is None:
        k_scale = q_scale
    if k_w is None:
        k_w = q_w
    return (rows_dq(q_acc, freqs_cis, q_scale, epsilon, x_scale, q_w, split_half),
            rows_dq(k_acc, freqs_cis, k_scale, epsilon, x_scale, k_w, split_half))


# ------------------------------------------------------- positions on several axes
class AxisFrequencies(NamedTuple):
    """How the pairs of a head turn; both on the heads' device."""
    inv_freq: torch.Tensor    # fp64 [P] radians a position
    axis: torch.Tensor        # int32 [P] the axis whose position counts


def axis_frequencies(sections, base=10000.0, *, shared=True, interleaved=False, device="cuda"):
    """Frequencies for ``len(sections)`` axes with ``sections[a]`` pairs each, P in all.

    ``shared``: one run ``base ** (-j / P)`` over all pairs, each turned by its axis's
    position; otherwise every axis has a run of its own, ``base ** (-i / sections[a])``.
    The axes' pairs follow each other, or with ``interleaved`` take turns while an axis has
    pairs left.  Other frequencies (scaled ones, say) are an :class:`AxisFrequencies` of
    their own."""
    sections = [int(n) for n in sections]
    if not 1 <= len(sections) <= MAX_AXES or min(sections) < 0 or not 1 <= sum(sections) <= MAX_PAIRS:
        raise ValueError(f"sections must be 1..{MAX_AXES} numbers of pairs, 1..{MAX_PAIRS} in all, "
                         f"got {sections}")
    if not base > 0:
        raise ValueError(f"base must be positive, got {base!r}")
    pairs = [(a, i) for a, n in enumerate(sections) for i in range(n)]
    if interleaved:
        pairs.sort(key=lambda p: (p[1], p[0]))
    exponent = [j / len(pairs) if shared else i / sections[a] for j, (a, i) in enumerate(pairs)]
    inv = torch.tensor([float(base) ** -x for x in exponent], dtype=torch.float64)
    axis = torch.tensor([a for a, _ in pairs], dtype=torch.int32)
    return AxisFrequencies(inv.to(device), axis.to(device))


def _strides(x, out):
    return (ctypes.c_int64 * 6)(*x.stride()[:3], *out.stride()[:3])


def _heads(x):
    """``x`` [B, S, H, D] with a contiguous head dimension"""
    x = x.resolve_neg()
    return x if x.stride(3) == 1 or x.shape[3] == 1 else x.contiguous()


def _like(x):
    """An empty result in x's layout if that is dense, else contiguous"""
    out = torch.empty_like(x)
    return out if out.stride(3) == 1 else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _turn(q, k, positions, frequencies, inverse, split_half):
    """The heads of q and, unless None, k by their angles"""
    q = _heads(q)
    oq = _like(q)
    ok = None
    if k is not None:
        k = _heads(k)
        ok = _like(k)
    b, s, _, d = q.shape
    if not b * s:
        return oq, ok
    first = positions.stride(0), 0 if positions.dim() == 2 else positions.stride(1), positions.stride(-1)
    lib = L._lib()
    with L._on(q.device):
        if lib.xpuint8_rope_axes_stream(
                L._stream(q.device), q.data_ptr(), oq.data_ptr(), _strides(q, oq), q.shape[2],
                _opt(k), _opt(ok), None if k is None else _strides(k, ok),
                0 if k is None else k.shape[2], TYPES[q.dtype], positions.data_ptr(),
                POSITION_TYPES[positions.dtype], (ctypes.c_int64 * 3)(*first), positions.shape[0],
                frequencies.inv_freq.data_ptr(), frequencies.axis.data_ptr(),
                frequencies.axis.numel(), int(inverse), int(split_half), b, s, d) != 0:
            L._err(lib, "rope.rotate_axes")
    return oq, ok


class _TurnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, inv_freq, axis, split_half):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, inv_freq, axis)
        ctx.split_half = split_half
        oq, ok = _turn(q, k, positions, AxisFrequencies(inv_freq, axis), False, split_half)
        return oq if k is None else (oq, ok)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk=None):
        L.check_backward(dq, dk)
        positions, *frequencies = ctx.saved_tensors
        frequencies = AxisFrequencies(*frequencies)
        dq = dq if ctx.needs_input_grad[0] else None
        dk = dk if ctx.needs_input_grad[1] else None
        if dq is None:
            if dk is not None:
                dk, _ = _turn(dk, None, positions, frequencies, True, ctx.split_half)
        else:
            dq, dk = _turn(dq, dk, positions, frequencies, True, ctx.split_half)
        return dq, dk, None, None, None, None


def rotate_axes(q, k, positions, frequencies, *, split_half=True):
    """q [B, S, Hq, D] and k [B, S, Hk, D] (or None) turned by their positions: pair j by
    ``positions[axis[j], b, s] * inv_freq[j]``, (a, b) becoming (a cos - b sin,
    b cos + a sin).  Returns (q, k) in their type (bf16, fp16 or fp32) and layout (a layout
    with gaps: contiguous), with gradients to both.

    ``positions`` [A, B, S], or [A, S] for all of the batch: int32, int64 or fp32.  Angles
    are reduced in fp64, to 2^-51 of themselves: closer than fp32 tells apart up to 10^8
    radians, less beyond.  ``frequencies`` is an :class:`AxisFrequencies` of P
    pairs (:func:`axis_frequencies`); a pair whose axis is not in 0..A-1 is not turned.
    Pairs are the elements j and j + P with ``split_half``, else 2j and 2j + 1; those past
    2 P stay as they are.  Strides are free but for a contiguous head dimension (others are
    copied): a [B, H, S, D] tensor goes in as ``x.transpose(1, 2)``.  Positions and
    frequencies have no gradient, and ones that need one are refused."""
    if L.HOST is not None and type(frequencies) is AxisFrequencies:
        r = L.HOST.rotate_axes(q, k, positions, frequencies, split_half)
        if r is not None:
            return r
    _check_float(q, "q")
    if q.dim() != 4 or 0 in q.shape[2:]:
        raise ValueError(f"q must be [B, S, H, D], got {tuple(q.shape)}")
    if k is not None:
        _check_float(k, "k")
        if k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3] or not k.shape[2]:
            raise ValueError(f"k must be [{q.shape[0]}, {q.shape[1]}, H, {q.shape[3]}], got "
                             f"{tuple(k.shape)}")
        if k.dtype != q.dtype or k.device != q.device:
            raise TypeError(f"k is {k.dtype} on {k.device} but q is {q.dtype} on {q.device}")
    if q.shape[2] + (0 if k is None else k.shape[2]) > MAX_HEADS or q.shape[3] > MAX_HEAD_DIM:
        raise ValueError(f"at most {MAX_HEADS} heads of {MAX_HEAD_DIM} are supported")
    if not isinstance(frequencies, AxisFrequencies):
        raise TypeError(f"frequencies must be a rope.AxisFrequencies, got "
                        f"{type(frequencies).__name__}")
    for t, name, dtype in zip(frequencies, AxisFrequencies._fields, (torch.float64, torch.int32)):
        if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != 1 or not t.is_contiguous():
            raise TypeError(f"frequencies.{name} must be a contiguous {dtype} vector")
        if t.device != q.device:
            raise TypeError(f"frequencies.{name} is on {t.device} but q is on {q.device}")
    pairs = frequencies.axis.numel()
    if frequencies.inv_freq.numel() != pairs:
        raise ValueError("frequencies' tensors do not belong together")
    if not 1 <= pairs <= MAX_PAIRS or 2 * pairs > q.shape[3]:
        raise ValueError(f"frequencies of {pairs} pairs do not fit heads of {q.shape[3]} (at most "
                         f"{MAX_PAIRS} pairs)")
    if not isinstance(positions, torch.Tensor) or positions.dtype not in POSITION_TYPES:
        raise TypeError(f"positions must be an int32, int64 or float32 tensor, got "
                        f"{getattr(positions, 'dtype', type(positions).__name__)}")
    if positions.device != q.device:
        raise TypeError(f"positions is on {positions.device} but q is on {q.device}")
    if (positions.dim() not in (2, 3) or not 1 <= positions.shape[0] <= MAX_AXES
            or positions.shape[1:] not in (q.shape[:2], q.shape[1:2])):
        raise ValueError(f"positions must be [A, {q.shape[0]}, {q.shape[1]}] or [A, {q.shape[1]}] "
                         f"with 1..{MAX_AXES} axes, got {tuple(positions.shape)}")
    if torch.is_grad_enabled() and (positions.requires_grad or frequencies.inv_freq.requires_grad):
        raise ValueError("positions and frequencies get no gradient")
    wanted = _wants_grad(q, k, positions, frequencies.inv_freq)
    positions = positions.detach().resolve_neg()
    frequencies = AxisFrequencies(*(t.detach().resolve_neg() for t in frequencies))
    if wanted:
        _check_leaves(q, k)
        r = _TurnFn.apply(q, k, positions, *frequencies, bool(split_half))
        return (r, None) if k is None else r
    return _turn(q, k, positions, frequencies, False, bool(split_half))
