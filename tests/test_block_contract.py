"""The refusals of RMS norm, routing and rotary positions, without a device: each argument
error is raised before the library or a GPU is touched."""

import ctypes

import pytest
import torch

from xpu_kernels import int8, moe, norm, rope
from xpu_kernels.int8 import _lib as L

X, I32 = torch.zeros(4, 64), torch.int32
Q = torch.zeros(2, 3, 4, 16)
F = rope.axis_frequencies((8,), device="cpu")
POS = torch.zeros(1, 2, 3, dtype=I32)
Q8, S8, W8 = torch.zeros(4, 64, dtype=torch.int8), torch.ones(4), torch.zeros(32, 64, dtype=torch.int8)

CASES = [
    ("norm-type", lambda: norm.rms_norm(X.double()), TypeError, "float64"),
    ("norm-list", lambda: norm.rms_norm([1.0]), TypeError, "list"),
    ("norm-cpu", lambda: norm.rms_norm(X), TypeError, "GPU"),
    ("int8-cpu", lambda: norm.rms_norm_int8(X), TypeError, "GPU"),
    ("route-cpu", lambda: moe.route(X, 2), TypeError, "GPU"),
    ("route-type", lambda: moe.route(X.int(), 2), TypeError, "int32"),
    ("rope-cpu", lambda: rope.rotate_axes(Q, None, POS, F), TypeError, "GPU"),
    ("rope-type", lambda: rope.rotate_axes(Q.double(), None, POS, F), TypeError, "float64"),
    ("frequencies-none", lambda: rope.axis_frequencies(()), ValueError, "sections"),
    ("frequencies-zero", lambda: rope.axis_frequencies((0, 0)), ValueError, "sections"),
    ("frequencies-negative", lambda: rope.axis_frequencies((4, -1)), ValueError, "sections"),
    ("frequencies-many", lambda: rope.axis_frequencies((513,)), ValueError, "512"),
    ("frequencies-base", lambda: rope.axis_frequencies((4,), 0.0), ValueError, "base"),
    ("quantized-q", lambda: int8.linear_quantized(X, S8, W8, S8), TypeError, "q must"),
    ("quantized-w", lambda: int8.linear_quantized(Q8, S8, X, S8), TypeError, "w8"),
    ("quantized-k", lambda: int8.linear_quantized(Q8[:, :32], S8, W8, S8), ValueError, "K mismatch"),
    ("quantized-16", lambda: int8.linear_quantized(Q8[:, :8], S8, W8[:, :8], S8), ValueError, "16"),
    ("quantized-scale", lambda: int8.linear_quantized(Q8, S8.half(), W8, S8), TypeError, "float32"),
    ("quantized-scales", lambda: int8.linear_quantized(Q8, S8[:3], W8, S8), ValueError, "4 rows"),
    ("quantized-ws", lambda: int8.linear_quantized(Q8, S8, W8, torch.ones(31)), ValueError, "N=32"),
    ("quantized-bias", lambda: int8.linear_quantized(Q8, S8, W8, torch.ones(32), torch.ones(3)),
     ValueError, "bias"),
    ("quantized-cpu", lambda: int8.linear_quantized(Q8, S8, W8, torch.ones(32)), TypeError, "GPU"),
]


@pytest.mark.parametrize("call,error,match", [c[1:] for c in CASES], ids=[c[0] for c in CASES])
def test_refusals(call, error, match):
    with pytest.raises(error, match=match):
        call()


P, Z, ODD = ctypes.c_void_p(0x1000), ctypes.c_void_p(0), ctypes.c_void_p(0x1001)
B8 = ctypes.c_void_p(0x1008)
STRIDES = (ctypes.c_int64 * 6)(1, 1, 1, 1, 1, 1)


@pytest.fixture(scope="module")
def lib():
    path = L.library_path()
    assert path is not None, "libxpuint8.so is not built (run __graft_entry__.build())"
    return L.open_library(path)


def norm_args(**kw):
    a = dict(st=Z, x=P, type=0, ldx=64, ox=64, r=Z, ldr=0, outer_r=0, inner=1, w=P, wt=2, eps=1e-6, h=Z, y=P, M=4, K=64)
    return tuple({**a, **kw}.values())


def int8_args(**kw):
    a = dict(st=Z, x=P, type=0, ldx=256, ox=256, r=Z, ldr=0, outer_r=0, inner=1, w=P, wt=2, eps=1e-6, h=Z, q=P, s=P, rot=1, M=4,
             K=256)
    return tuple({**a, **kw}.values())


def grad_args(**kw):
    a = dict(st=Z, dy=P, type=0, ldy=64, oy=64, h=P, ldh=64, oh=64, w=P, wt=2, dh=Z, lddh=0, odh=0, inner=1, eps=1e-6, dx=P, dw=P,
             M=4, K=64, work=P, n=1 << 20)
    return tuple({**a, **kw}.values())


def rope_args(**kw):
    a = dict(st=Z, q=P, qo=P, qs=STRIDES, hq=4, k=P, ko=P, ks=STRIDES, hk=2, type=0, p=P, pt=0,
             ps=STRIDES, axes=3, f=P, axis=P, pairs=32, inv=0, split=1, B=2, S=3, D=64)
    return tuple({**a, **kw}.values())


def route_args(**kw):
    a = dict(st=Z, l=P, type=0, ld=64, b=Z, sig=0, groups=1, tg=1, ren=1, scale=1.0, ids=P, w=P, T=4,
             E=64, top=8)
    return tuple({**a, **kw}.values())


def route_grad_args(**kw):
    a = dict(st=Z, l=P, type=0, ld=64, ids=P, dw=P, sig=0, ren=1, scale=1.0, dl=P, T=4, E=64, top=8)
    return tuple({**a, **kw}.values())


@pytest.mark.parametrize("fn,args,code,substr", [
    ("rms_norm", norm_args(M=0), 2, "positive"), ("rms_norm", norm_args(K=0), 2, "positive"),
    ("rms_norm", norm_args(M=1 << 31), 4, "2^31"), ("rms_norm", norm_args(K=1 << 25, ox=1 << 25), 4, "2^24"),
    ("rms_norm", norm_args(type=3), 6, "type"), ("rms_norm", norm_args(wt=3), 6, "weight_type"),
    ("rms_norm", norm_args(ox=63), 2, "stride"), ("rms_norm", norm_args(r=P, outer_r=63, h=P), 2, "stride"),
    ("rms_norm", norm_args(eps=-1.0), 2, "eps"), ("rms_norm", norm_args(eps=float("nan")), 2, "eps"),
    ("rms_norm", norm_args(x=Z), 6, "null"), ("rms_norm", norm_args(x=ODD), 6, "aligned"),
    ("rms_norm", norm_args(r=P, outer_r=64), 6, "together"), ("rms_norm", norm_args(h=P), 6, "together"),
    ("rms_norm", norm_args(r=ODD, outer_r=64, h=P), 6, "aligned"),
    ("rms_norm", norm_args(r=P, outer_r=64, h=B8), 6, "16-byte"), ("rms_norm", norm_args(w=ODD), 6, "weight"),
    ("rms_norm", norm_args(y=Z), 6, "null"), ("rms_norm", norm_args(y=B8), 6, "16-byte"),
    ("rms_norm", norm_args(inner=0), 2, "inner"), ("rms_norm", norm_args(inner=3), 2, "divide"),
    ("rms_norm", norm_args(inner=2, ldx=63, ox=128), 2, "stride"), ("rms_norm", norm_args(inner=2, ox=-1), 2, "stride"),
    ("rms_norm_grad", grad_args(inner=3), 2, "divide"), ("rms_norm_grad", grad_args(inner=2, ldh=63), 2, "stride"),
    ("rms_norm_int8", int8_args(K=255), 3, "256"), ("rms_norm_int8", int8_args(rot=2), 2, "rotate"),
    ("rms_norm_int8", int8_args(q=Z), 6, "null"), ("rms_norm_int8", int8_args(s=B8), 6, "16-byte"),
    ("rms_norm_int8", int8_args(M=-1), 2, "positive"),
    ("rms_norm_grad", grad_args(M=0), 2, "positive"), ("rms_norm_grad", grad_args(type=-1), 6, "type"),
    ("rms_norm_grad", grad_args(oy=63), 2, "stride"), ("rms_norm_grad", grad_args(oh=63), 2, "stride"),
    ("rms_norm_grad", grad_args(dh=P, odh=63), 2, "stride"), ("rms_norm_grad", grad_args(dy=Z), 6, "null"),
    ("rms_norm_grad", grad_args(dh=ODD, odh=64), 6, "aligned"), ("rms_norm_grad", grad_args(dx=B8), 6, "16-byte"),
    ("rms_norm_grad", grad_args(w=Z), 6, "needs a weight"), ("rms_norm_grad", grad_args(work=Z), 6, "work"),
    ("rms_norm_grad", grad_args(n=4 * 64 - 1), 2, "workspace_size"),
    ("rope_axes", rope_args(B=0), 2, "positive"), ("rope_axes", rope_args(S=1 << 31), 4, "2^31"),
    ("rope_axes", rope_args(B=1 << 16, S=1 << 16), 4, "2^31"),
    ("rope_axes", rope_args(pairs=33), 2, "pairs"), ("rope_axes", rope_args(pairs=0), 2, "pairs"),
    ("rope_axes", rope_args(pairs=513, D=4096), 2, "512"), ("rope_axes", rope_args(D=4097), 4, "4096"),
    ("rope_axes", rope_args(axes=0), 2, "axes"), ("rope_axes", rope_args(axes=17), 2, "axes"),
    ("rope_axes", rope_args(type=4), 6, "type"), ("rope_axes", rope_args(pt=3), 6, "position_type"),
    ("rope_axes", rope_args(split=2), 2, "split_half"), ("rope_axes", rope_args(q=Z), 6, "null"),
    ("rope_axes", rope_args(f=Z), 6, "null"), ("rope_axes", rope_args(ko=Z), 6, "together"),
    ("rope_axes", rope_args(hq=0), 2, "heads"), ("rope_axes", rope_args(hk=0), 2, "heads"),
    ("rope_axes", rope_args(hq=65536), 2, "65536"), ("rope_axes", rope_args(q=ODD), 6, "aligned"),
    ("rope_axes", rope_args(ko=ODD), 6, "aligned"), ("rope_axes", rope_args(p=ODD), 6, "aligned"),
    ("rope_axes", rope_args(f=ctypes.c_void_p(0x1004)), 6, "aligned"),
    ("moe_route", route_args(T=0), 2, "tokens"), ("moe_route", route_args(E=1025, ld=1025), 2, "1..1024"),
    ("moe_route", route_args(top=65), 2, "top"), ("moe_route", route_args(E=4, top=5), 2, "top"),
    ("moe_route", route_args(type=3), 6, "type"), ("moe_route", route_args(ld=63), 2, "stride"),
    ("moe_route", route_args(sig=2), 2, "sigmoid"), ("moe_route", route_args(groups=3), 2, "divide"),
    ("moe_route", route_args(groups=65, E=65, ld=65), 2, "64"), ("moe_route", route_args(groups=8, tg=9), 2, "top_groups"),
    ("moe_route", route_args(groups=16, tg=1), 2, "hold top"), ("moe_route", route_args(ids=Z), 6, "null"),
    ("moe_route", route_args(l=ODD), 6, "aligned"), ("moe_route", route_args(b=ctypes.c_void_p(0x1002)), 6, "bias"),
    ("moe_route_grad", route_grad_args(dl=Z), 6, "null"), ("moe_route_grad", route_grad_args(ren=-1), 2, "renormalize"),
    ("moe_route_grad", route_grad_args(dl=ODD), 6, "aligned"), ("moe_route_grad", route_grad_args(T=1 << 31), 2, "tokens"),
])
def test_library_refusals(lib, fn, args, code, substr):
    rc = getattr(lib, f"xpuint8_{fn}_stream")(*args)
    msg = lib.xpuint8_last_error().decode()
    assert rc == code and substr in msg, (rc, msg)


def test_gradient_workspace(lib):
    size = lib.xpuint8_rms_norm_grad_workspace_size
    assert size(0, 64) == size(4, 0) == size(1, (1 << 24) + 1) == -1
    assert size(1, 64) == 64 * 4 and size(1 << 20, 4096) == 512 * 4096 * 4
