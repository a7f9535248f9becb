"""Mixture-of-experts routing on gfx950: tokens sorted by expert and back, with
the weights applied, their gradients, and an FFN of MXFP4 experts.

    routing = moe.sort(expert_ids, n_experts)     # expert_ids [T, top], integers
    xs = moe.dispatch(x, routing)                 # [T, D] -> [T*top, D], by expert
    ...                                           # the experts, on their rows
    y = moe.combine(zs, routing, weights)         # [T*top, D] -> [T, D]

A slot whose id is outside [0, n_experts) belongs to no expert (a token over an
expert's capacity, an expert of another rank): it is sorted last, its rows are
zeros, and it adds nothing to its token and gets no gradient.  The sort is stable
and every sum has a fixed order, so results are the same from call to call.  All
of it runs in ``libxpuint8.so`` on torch's current stream without synchronising
(no count reaches the host); there is no counterpart in the reference.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import mxfp4
from .int8 import _lib as L
from .mxfp4 import TYPES, _check_float, _opt, _rows, _wants_grad, _work

__all__ = ["Routing", "combine", "dispatch", "ffn", "sort"]

MAX_EXPERTS = 1024


class Routing(NamedTuple):
    """Where each slot went; all int32 on the tokens' device."""
    order: torch.Tensor       # [T*top] the slot (t * top + j) of each sorted row
    position: torch.Tensor    # [T, top] the sorted row of each slot
    rows: torch.Tensor        # [T*top] the token of each sorted row
    offsets: torch.Tensor     # [E + 1] the first row of each expert; past [E]: no expert


def _check_routing(routing, device):
    if not isinstance(routing, Routing):
        raise TypeError(f"routing must be a moe.Routing, got {type(routing).__name__}")
    n = routing.order.numel()
    for t, name in zip(routing, Routing._fields):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or not t.is_contiguous():
            raise TypeError(f"routing.{name} must be a contiguous int32 tensor")
        if t.device != device:
            raise TypeError(f"routing.{name} is on {t.device} but the rows are on {device}")
    if (routing.position.dim() != 2 or routing.position.numel() != n or routing.rows.numel() != n
            or routing.offsets.numel() < 2):
        raise ValueError("routing's tensors do not belong together")


def sort(expert_ids, n_experts):
    """Sort the slots of ``expert_ids`` [T, top] (int32 or int64) by expert, stably."""
    if L.HOST is not None:
        r = L.HOST.moe_sort(expert_ids, n_experts)
        if r is not None:
            return Routing._make(r)
    if not isinstance(expert_ids, torch.Tensor) or expert_ids.dtype not in (torch.int32,
                                                                          torch.int64):
        raise TypeError(f"expert_ids must be an int32 or int64 tensor, got "
                        f"{getattr(expert_ids, 'dtype', type(expert_ids).__name__)}")
    if expert_ids.dim() != 2 or expert_ids.shape[1] < 1:
        raise ValueError(f"expert_ids must be [T, top], got {tuple(expert_ids.shape)}")
    if not 1 <= n_experts <= MAX_EXPERTS:
        raise ValueError(f"n_experts must be 1..{MAX_EXPERTS}, got {n_experts}")
    if expert_ids.device.type != "cuda":
        raise TypeError(f"expected a GPU (ROCm) tensor, got {expert_ids.device}")
    ids = expert_ids.contiguous()
    t, top = ids.shape
    # one allocation for the four results
    s = t * top
    buf = torch.empty(3 * s + n_experts + 1, dtype=torch.int32, device=ids.device)
    order, position, rows, offsets = buf.split((s, s, s, n_experts + 1))
    routing = Routing(order, position.view(t, top), rows, offsets)
    if not t:
        offsets.zero_()
        return routing
    lib = L._lib()
    need = lib.xpuint8_moe_sort_workspace_size(t, top, n_experts)
    work = _work(need, ids)
    if lib.xpuint8_moe_sort_stream(L._stream(ids.device), ids.data_ptr(),
                                   1 if ids.dtype == torch.int64 else 0, order.data_ptr(),
                                   position.data_ptr(), rows.data_ptr(), offsets.data_ptr(), t,
                                   top, n_experts, _opt(work), need) != 0:
        L._err(lib, "moe.sort")
    return routing


def _dispatch(x, routing):
    t, top = routing.position.shape
    d = x.shape[1]
    out = torch.empty((t * top, d), dtype=x.dtype, device=x.device)
    if t and d:
        x2, ld = _rows(x)
        lib = L._lib()
        if lib.xpuint8_moe_dispatch_stream(L._stream(x.device), x2.data_ptr(), TYPES[x.dtype], ld,
                                           routing.position.data_ptr(),
                                           routing.offsets.data_ptr(), out.data_ptr(), t, top,
                                           routing.offsets.numel() - 1, d) != 0:
            L._err(lib, "moe.dispatch")
    return out


def _combine(z, routing, weights, out_dtype):
    t, top = routing.position.shape
    d = z.shape[1]
    out = torch.empty((t, d), dtype=out_dtype, device=z.device)
    if t and d:
        z2, ld = _rows(z)
        lib = L._lib()
        if lib.xpuint8_moe_combine_stream(L._stream(z.device), z2.data_ptr(), TYPES[z.dtype], ld,
                                          routing.position.data_ptr(),
                                          routing.offsets.data_ptr(), _opt(weights),
                                          out.data_ptr(), TYPES[out_dtype], t, top,
                                          routing.offsets.numel() - 1, d) != 0:
            L._err(lib, "moe.combine")
    return out


class _DispatchFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, routing):
        ctx.save_for_backward(*routing)
        return _dispatch(x, routing)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dxs):
        return _combine(dxs, Routing(*ctx.saved_tensors), None, dxs.dtype), None


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, weights, routing):
        ctx.save_for_backward(z, weights, *routing)
        return _combine(z, routing, weights, z.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        z, weights, *routing = ctx.saved_tensors
        routing = Routing(*routing)
        t, top = routing.position.shape
        d = z.shape[1]
        dz = torch.empty((t * top, d), dtype=z.dtype, device=z.device)
        dweights = torch.empty((t, top), dtype=torch.float32, device=z.device)
        if not t or not d:
            return dz, dweights.zero_(), None
        dy2, ldy = _rows(dy)
        z2, ldz = _rows(z)
        lib = L._lib()
        if lib.xpuint8_moe_combine_grad_stream(
                L._stream(z.device), dy2.data_ptr(), TYPES[z.dtype], ldy, z2.data_ptr(), ldz,
                routing.position.data_ptr(), routing.offsets.data_ptr(), weights.data_ptr(),
                dz.data_ptr(), dweights.data_ptr(), t, top, routing.offsets.numel() - 1, d) != 0:
            L._err(lib, "moe.combine (gradient)")
        return dz, dweights, None


def dispatch(x, routing):
    """x [T, D] -> [T*top, D]: each token's row at each of its slots' places, in
    the experts' order; zeros in the rows of no expert.  The gradient sums a
    token's rows in fp32."""
    if L.HOST is not None and type(routing) is Routing:
        r = L.HOST.moe_dispatch(x, routing)
        if r is not None:
            return r
    _check_float(x, "x")
    _check_routing(routing, x.device)
    if x.dim() != 2 or x.shape[0] != routing.position.shape[0]:
        raise ValueError(f"x must be [{routing.position.shape[0]}, D], got {tuple(x.shape)}")
    if _wants_grad(x):
        return _DispatchFn.apply(x, routing)
    return _dispatch(x, routing)


def combine(z, routing, weights):
    """z [T*top, D] in the experts' order -> [T, D]: each token's rows times
    ``weights`` [T, top] (used in fp32), summed in fp32 in slot order.  Gradients
    reach z and weights."""
    if L.HOST is not None and type(routing) is Routing:
        r = L.HOST.moe_combine(z, routing, weights)
        if r is not None:
            return r
    _check_float(z, "z")
    _check_routing(routing, z.device)
    t, top = routing.position.shape
    if z.dim() != 2 or z.shape[0] != t * top:
        raise ValueError(f"z must be [{t * top}, D], got {tuple(z.shape)}")
    _check_float(weights, "weights")
    if weights.shape != (t, top):
        raise ValueError(f"weights must be [{t}, {top}], got {tuple(weights.shape)}")
    if weights.device != z.device:
        raise TypeError(f"weights is on {weights.device} but z is on {z.device}")
    weights = weights.float().resolve_neg().contiguous()
    if _wants_grad(z, weights):
        return _CombineFn.apply(z, weights, routing)
    return _combine(z, routing, weights, z.dtype)


def ffn(x, expert_ids, weights, up, down):
    """A mixture of gated MXFP4 experts: each token [T, D] through its experts'
    ``down(silu(gate) * up)``, weighted and summed.

    ``up`` is (codes [E, 2F, D/2], scales), the gate's F rows first; ``down``
    (codes [E, D, F/2], scales).  Sort, the gathering up-projection, the
    activation in fp32, the down-projection and the weighted sum; gradients reach
    x and weights."""
    routing = sort(expert_ids, up[0].shape[0])
    h = mxfp4.grouped_linear(x, *up, routing, gather=True)
    gate, value = h.chunk(2, dim=-1)
    h = (torch.nn.functional.silu(gate.float()) * value.float()).to(x.dtype)
    return combine(mxfp4.grouped_linear(h, *down, routing), routing, weights)
