"""MXFP4 linears on gfx950: microscaled 4-bit quantization, the product of
4-bit activations with a 4-bit weight, the experts' products, and their gradients.

A tensor [.., K] (K a multiple of 32) in MXFP4 is two uint8 tensors:

* ``codes`` [.., K/2], element 2i in the low half of byte i;
* ``scales`` [.., ``scale_width(K)``], the power of two of each block of 32
  values (its exponent + 127, 255 for a NaN block), a row padded to whole groups
  of 16 blocks (512 values).  :func:`pad_scales` makes it from a checkpoint's
  [.., K/32].

A block's exponent is ``clamp(floor(log2 amax) - 2, -127, 127)``; values round to
nearest even on {0, .5, 1, 1.5, 2, 3, 4, 6} and saturate at 6; a block with an
infinity or NaN reads back as NaNs.

    codes, scales = mxfp4.quantize(w)                 # bf16, fp16 or fp32 [N, K]
    y = mxfp4.linear(x, codes, scales, bias)          # [.., K] -> [.., N], x's type

The weight is frozen; gradients reach ``x`` (straight through its quantization)
and ``bias``; forward-mode derivatives are refused.  Everything runs in ``libxpuint8.so`` on torch's current stream,
without synchronising; there is no counterpart in the reference.
"""

from __future__ import annotations

import torch
from torch.autograd.forward_ad import unpack_dual

from .int8 import _lib as L

__all__ = ["dequantize", "grouped_linear", "linear", "pad_scales", "quantize", "scale_width"]

#: element types by the library's number
TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
BLOCK = 32


def scale_width(k: int) -> int:
    """Bytes of a row of scales of ``k`` values."""
    if k <= 0 or k % BLOCK:
        raise ValueError(f"K={k} is not a positive multiple of the MXFP4 block ({BLOCK})")
    return -(-k // 512) * 16


def pad_scales(scales):
    """Scales [.., K/32] as the kernels read them: [.., scale_width(K)], a copy
    only if the rows need padding."""
    if scales.dtype != torch.uint8:
        raise TypeError(f"scales must be uint8, got {scales.dtype}")
    n = scales.shape[-1]
    width = scale_width(n * BLOCK)
    if width == n:
        return scales
    return torch.nn.functional.pad(scales, (0, width - n), value=127)


def _check_float(t, name):
    if not isinstance(t, torch.Tensor) or t.dtype not in TYPES:
        raise TypeError(f"{name} must be a bfloat16, float16 or float32 tensor, got "
                        f"{getattr(t, 'dtype', type(t).__name__)}")
    if t.device.type != "cuda":
        raise TypeError(f"expected a GPU (ROCm) tensor, got {t.device}")


def _wants_grad(*tensors):
    """Whether any of the tensors (or Nones) needs a gradient; a forward-mode tangent,
    which no operator here carries on, is refused."""
    tensors = [t for t in tensors if t is not None]
    if any(unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("the operators of norm, mxfp4, moe and rope have no "
                                  "forward-mode derivative")
    return torch.is_grad_enabled() and any(t.requires_grad for t in tensors)


def _check_leaves(*tensors):
    """Refuse a captured call whose backward pass would break the capture."""
    if L.HOST is not None:
        L.HOST.check_leaves(*tensors)


def _check_pair(codes, scales, lead=None):
    """The K behind codes and scales, both on the GPU and of matching shapes."""
    for t, name in ((codes, "codes"), (scales, "scales")):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8:
            raise TypeError(f"{name} must be a uint8 tensor, got "
                            f"{getattr(t, 'dtype', type(t).__name__)}")
    if codes.dim() < 1 or codes.dim() != scales.dim() or codes.shape[:-1] != scales.shape[:-1]:
        raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not "
                         f"belong together")
    if lead is not None and codes.dim() != lead:
        raise ValueError(f"codes must have {lead} dimensions, got {tuple(codes.shape)}")
    k = codes.shape[-1] * 2
    if scales.shape[-1] != scale_width(k):
        raise ValueError(f"scales must have {scale_width(k)} bytes a row for K={k}, got "
                         f"{scales.shape[-1]} (see pad_scales)")
    if codes.device.type != "cuda":
        raise TypeError(f"expected a GPU (ROCm) tensor, got {codes.device}")
    if scales.device != codes.device:
        raise TypeError(f"scales is on {scales.device} but codes is on {codes.device}")
    return k


def _rows(x):
    """``x`` [.., K] as rows with a stride: (tensor [M, K] or a view, row stride); a
    sign that is a flag of the view is applied."""
    x2 = x.resolve_neg().reshape(-1, x.shape[-1])
    if x2.stride(-1) != 1 or (x2.shape[0] > 1 and x2.stride(0) < x2.shape[1]):
        x2 = x2.contiguous()
    ld = x2.stride(0) if x2.shape[0] > 1 else x2.shape[1]
    return x2, ld


def _work(nbytes, like):
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes > 0 else None


def _opt(t):
    return None if t is None else t.data_ptr()


def quantize(x):
    """x [.., K] (bf16, fp16 or fp32) -> (codes uint8 [.., K/2], scales uint8
    [.., scale_width(K)])."""
    if L.HOST is not None:
        r = L.HOST.mx_quantize(x)
        if r is not None:
            return r
    _check_float(x, "x")
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    k = x.shape[-1]
    width = scale_width(k)
    x2, ld = _rows(x.detach())
    codes = torch.empty((*x.shape[:-1], k // 2), dtype=torch.uint8, device=x.device)
    scales = torch.empty((*x.shape[:-1], width), dtype=torch.uint8, device=x.device)
    if x2.shape[0]:
        lib = L._lib()
        if lib.xpuint8_mxfp4_quantize_stream(L._stream(x.device), x2.data_ptr(), TYPES[x.dtype],
                                             ld, codes.data_ptr(), scales.data_ptr(),
                                             x2.shape[0], k) != 0:
            L._err(lib, "mxfp4.quantize")
    return codes, scales


def dequantize(codes, scales, dtype=torch.bfloat16):
    """What codes and scales stand for, [.., K] in ``dtype`` (bf16 and fp32 hold
    every value; fp16 turns what is beyond its range into infinities)."""
    if L.HOST is not None and dtype in TYPES:
        r = L.HOST.mx_dequantize(codes, scales, TYPES[dtype])
        if r is not None:
            return r
    k = _check_pair(codes, scales)
    if dtype not in TYPES:
        raise TypeError(f"dtype must be bfloat16, float16 or float32, got {dtype}")
    codes, scales = L._c(codes), L._c(scales)
    out = torch.empty((*codes.shape[:-1], k), dtype=dtype, device=codes.device)
    m = codes.numel() // (k // 2)
    if m:
        lib = L._lib()
        if lib.xpuint8_mxfp4_dequantize_stream(L._stream(codes.device), codes.data_ptr(),
                                               scales.data_ptr(), out.data_ptr(), TYPES[dtype],
                                               m, k) != 0:
            L._err(lib, "mxfp4.dequantize")
    return out


def _check_weight(x, codes, scales, dims):
    _check_float(x, "x")
    k = _check_pair(codes, scales, dims)
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"x has {x.shape[-1] if x.dim() else 0} columns but the weight has K={k}")
    if codes.device != x.device:
        raise TypeError(f"the weight is on {codes.device} but x is on {x.device}")
    return k


def _linear(x, codes, scales, bias):
    n, k = codes.shape[0], x.shape[-1]
    y = torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
    x2, ld = _rows(x)
    m = x2.shape[0]
    if m and n:
        lib = L._lib()
        need = lib.xpuint8_mxfp4_linear_workspace_size(m, n, k)
        work = _work(need, x)
        if lib.xpuint8_mxfp4_linear_stream(L._stream(x.device), x2.data_ptr(), TYPES[x.dtype], ld,
                                           codes.data_ptr(), scales.data_ptr(), _opt(bias),
                                           0 if bias is None else TYPES[bias.dtype], y.data_ptr(),
                                           m, n, k, _opt(work), need) != 0:
            L._err(lib, "mxfp4.linear")
    return y


def _dx(dy, codes, scales, offsets, out_dtype):
    """dy [.., N] times the (experts') weight, [R, K]."""
    n, k = codes.shape[-2], codes.shape[-1] * 2
    dy2, ld = _rows(dy)
    r = dy2.shape[0]
    dx = torch.empty((r, k), dtype=out_dtype, device=dy.device)
    if not n:
        return dx.zero_()
    if r:
        lib = L._lib()
        e = 0 if offsets is None else offsets.numel() - 1
        need = lib.xpuint8_mxfp4_dx_workspace_size_of(dy2.data_ptr(), TYPES[dy2.dtype], ld,
                                                      TYPES[out_dtype], r, e, n, k)
        work = _work(need, dy2)
        if lib.xpuint8_mxfp4_dx_stream(L._stream(dy.device), dy2.data_ptr(), TYPES[dy2.dtype], ld,
                                       codes.data_ptr(), scales.data_ptr(), _opt(offsets), e,
                                       dx.data_ptr(), TYPES[out_dtype], r, n, k, _opt(work),
                                       need) != 0:
            L._err(lib, "mxfp4 dx")
    return dx


def _dbias(dy, dtype):
    """The column sums of dy [.., N] in fp32, rounded once to ``dtype``."""
    dy2, ld = _rows(dy)
    m, n = dy2.shape
    out = torch.empty((n,), dtype=dtype, device=dy.device)
    if not m:
        return out.zero_()
    lib = L._lib()
    need = lib.xpuint8_mxfp4_dbias_workspace_size(m, n)
    work = _work(need, dy2)
    if lib.xpuint8_mxfp4_dbias_stream(L._stream(dy.device), dy2.data_ptr(), TYPES[dy2.dtype], ld,
                                      out.data_ptr(), TYPES[dtype], m, n, _opt(work), need) != 0:
        L._err(lib, "mxfp4 bias gradient")
    return out


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, codes, scales, bias):
        ctx.save_for_backward(codes, scales)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return _linear(x, codes, scales, bias)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        L.check_backward(dy)
        codes, scales = ctx.saved_tensors
        dx = dbias = None
        if ctx.needs_input_grad[0]:
            dx = _dx(dy, codes, scales, None, dy.dtype).reshape(*dy.shape[:-1], codes.shape[-1] * 2)
        if ctx.needs_input_grad[3]:
            dbias = _dbias(dy, ctx.bias_dtype)
        return dx, None, None, dbias


def linear(x, codes, scales, bias=None):
    """``xq @ wq.T + bias``: x [.., K] quantized to MXFP4 in the call, the weight
    codes [N, K/2] and scales [N, scale_width(K)]; fp32 sums rounded once to x's
    type.  ``bias`` [N] is bf16, fp16 or fp32.  Gradients: dx = dy @ wq, straight
    through x's quantization, and for the bias dy's column sums in fp32, rounded once to
    the bias's type; the weight has none."""
    if L.HOST is not None:
        r = L.HOST.mx_linear(x, codes, scales, bias)
        if r is not None:
            return r
    _check_weight(x, codes, scales, 2)
    codes, scales = L._c(codes), L._c(scales)
    if bias is not None:
        _check_float(bias, "bias")
        if bias.shape != (codes.shape[0],):
            raise ValueError(f"bias must have shape ({codes.shape[0]},), got {tuple(bias.shape)}")
        if bias.device != x.device:
            raise TypeError(f"bias is on {bias.device} but x is on {x.device}")
        bias = bias.resolve_neg().contiguous()
    if _wants_grad(x, bias):
        return _LinearFn.apply(x, codes, scales, bias)
    return _linear(x, codes, scales, bias)


def _grouped(x, codes, scales, routing, gather):
    e, n = codes.shape[:2]
    k = x.shape[-1]
    r = routing.order.numel()
    y = torch.empty((r, n), dtype=x.dtype, device=x.device)
    x2, ld = _rows(x)
    if r and n:
        lib = L._lib()
        need = lib.xpuint8_mxfp4_grouped_linear_workspace_size(r, x2.shape[0], e, n, k)
        work = _work(need, x)
        if lib.xpuint8_mxfp4_grouped_linear_stream(
                L._stream(x.device), x2.data_ptr(), TYPES[x.dtype], ld,
                routing.rows.data_ptr() if gather else None, x2.shape[0], codes.data_ptr(),
                scales.data_ptr(), routing.offsets.data_ptr(), e, y.data_ptr(), r, n, k,
                _opt(work), need) != 0:
            L._err(lib, "mxfp4.grouped_linear")
    return y


class _GroupedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, codes, scales, routing, gather):
        ctx.save_for_backward(codes, scales, *routing)
        ctx.gather = gather
        return _grouped(x, codes, scales, routing, gather)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        from . import moe
        L.check_backward(dy)
        codes, scales, *routing = ctx.saved_tensors
        routing = moe.Routing(*routing)
        if not ctx.gather:
            return _dx(dy, codes, scales, routing.offsets, dy.dtype), None, None, None, None
        # a token's rows are summed in fp32 and rounded once
        dxs = _dx(dy, codes, scales, routing.offsets, torch.float32)
        return moe._combine(dxs, routing, None, dy.dtype), None, None, None, None


def grouped_linear(x, codes, scales, routing, gather=False):
    """The experts' products over rows sorted by expert (``moe.sort``): row i of
    expert e is ``xq[i] @ wq[e].T``, rows of no expert are zeros.

    ``codes`` [E, N, K/2] and ``scales`` [E, N, scale_width(K)]; x [T*top, K] in
    the sorted order (``moe.dispatch``), or with ``gather`` the tokens themselves,
    [T, K], each quantized once and read by every row that is its.  Returns
    [T*top, N] in x's type; the gradient reaches x."""
    from . import moe
    if L.HOST is not None and type(routing) is moe.Routing:
        r = L.HOST.mx_grouped(x, codes, scales, routing, gather)
        if r is not None:
            return r
    _check_weight(x, codes, scales, 3)
    moe._check_routing(routing, x.device)
    if routing.offsets.numel() != codes.shape[0] + 1:
        raise ValueError(f"the routing has {routing.offsets.numel() - 1} experts but the weight "
                         f"has {codes.shape[0]}")
    want = routing.position.shape[0] if gather else routing.order.numel()
    if x.dim() != 2 or x.shape[0] != want:
        raise ValueError(f"x must be [{want}, K] ({'tokens' if gather else 'sorted rows'}), got "
                         f"{tuple(x.shape)}")
    codes, scales = L._c(codes), L._c(scales)
    if _wants_grad(x):
        return _GroupedFn.apply(x, codes, scales, routing, bool(gather))
    return _grouped(x, codes, scales, routing, gather)
