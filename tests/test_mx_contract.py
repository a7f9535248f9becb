"""The refusals of the MXFP4 and mixture-of-experts operators, without a device: each
argument error is raised before the library or a GPU is touched."""

import ctypes

import pytest
import torch

import oracle.mxfp4 as O
from xpu_kernels import moe, mxfp4
from xpu_kernels.int8 import _lib as L

BF16, U8, I32 = torch.bfloat16, torch.uint8, torch.int32


def pair(n=8, k=64):
    return torch.zeros(n, k // 2, dtype=U8), torch.full((n, mxfp4.scale_width(k)), 127, dtype=U8)


@pytest.mark.parametrize("k,width", [(32, 16), (512, 16), (544, 32), (1280, 48), (4096, 128)])
def test_scale_width(k, width):
    assert mxfp4.scale_width(k) == width == O.scale_width(k)


@pytest.mark.parametrize("k", [0, -32, 16, 33, 100])
def test_scale_width_refuses(k):
    with pytest.raises(ValueError, match="32"):
        mxfp4.scale_width(k)


def test_pad_scales():
    s = torch.arange(40, dtype=U8).repeat(3, 1)
    p = mxfp4.pad_scales(s)
    assert p.shape == (3, 48) and torch.equal(p[:, :40], s) and (p[:, 40:] == 127).all()
    full = torch.zeros(3, 16, dtype=U8)
    assert mxfp4.pad_scales(full) is full
    with pytest.raises(TypeError, match="uint8"):
        mxfp4.pad_scales(torch.zeros(3, 16))


CASES = [
    ("quantize-int", lambda: mxfp4.quantize(torch.zeros(4, 64, dtype=I32)), TypeError, "bfloat16"),
    ("quantize-double", lambda: mxfp4.quantize(torch.zeros(4, 64).double()), TypeError, "float64"),
    ("quantize-list", lambda: mxfp4.quantize([1.0]), TypeError, "list"),
    ("quantize-cpu", lambda: mxfp4.quantize(torch.zeros(4, 64)), TypeError, "GPU"),
    ("dequantize-type", lambda: mxfp4.dequantize(torch.zeros(4, 32), pair()[1]), TypeError, "uint8"),
    ("dequantize-rows", lambda: mxfp4.dequantize(pair(8)[0], pair(7)[1]), ValueError, "belong"),
    ("dequantize-width", lambda: mxfp4.dequantize(pair()[0], pair()[1][:, :2]), ValueError,
     "pad_scales"),
    ("dequantize-k", lambda: mxfp4.dequantize(torch.zeros(4, 8, dtype=U8), pair(4)[1]), ValueError,
     "32"),
    ("dequantize-cpu", lambda: mxfp4.dequantize(*pair()), TypeError, "GPU"),
    ("linear-cpu", lambda: mxfp4.linear(torch.zeros(2, 64, dtype=BF16), *pair()), TypeError, "GPU"),
    ("linear-x-type", lambda: mxfp4.linear(torch.zeros(2, 64, dtype=torch.int8), *pair()),
     TypeError, "int8"),
    ("sort-float", lambda: moe.sort(torch.zeros(2, 2), 4), TypeError, "int32"),
    ("sort-dims", lambda: moe.sort(torch.zeros(4, dtype=I32), 4), ValueError, "top"),
    ("sort-no-slots", lambda: moe.sort(torch.zeros(4, 0, dtype=I32), 4), ValueError, "top"),
    ("sort-experts", lambda: moe.sort(torch.zeros(4, 2, dtype=I32), 0), ValueError, "1..1024"),
    ("sort-many", lambda: moe.sort(torch.zeros(4, 2, dtype=I32), 1025), ValueError, "1..1024"),
    ("sort-cpu", lambda: moe.sort(torch.zeros(4, 2, dtype=I32), 4), TypeError, "GPU"),
    ("dispatch-cpu", lambda: moe.dispatch(torch.zeros(4, 8), None), TypeError, "GPU"),
    ("combine-type", lambda: moe.combine(torch.zeros(4, 8, dtype=I32), None, None), TypeError,
     "bfloat16"),
]


@pytest.mark.parametrize("call,kind,text", [c[1:] for c in CASES], ids=[c[0] for c in CASES])
def test_refusals(call, kind, text):
    with pytest.raises(kind, match=text):
        call()


@pytest.fixture(scope="module")
def lib():
    path = L.library_path()
    assert path is not None, "libxpuint8.so is not built (run __graft_entry__.build())"
    return L.open_library(path)


P, Z, ODD = ctypes.c_void_p(0x1000), ctypes.c_void_p(0), ctypes.c_void_p(0x1008)


@pytest.mark.parametrize("fn,args,code,substr", [
    ("mxfp4_quantize_stream", (Z, P, 0, 64, P, P, 0, 64), 2, "positive"),
    ("mxfp4_quantize_stream", (Z, P, 0, 64, P, P, 4, 48), 3, "32"),
    ("mxfp4_quantize_stream", (Z, P, 3, 64, P, P, 4, 64), 6, "bf16"),
    ("mxfp4_quantize_stream", (Z, P, 0, 63, P, P, 4, 64), 2, "stride"),
    ("mxfp4_quantize_stream", (Z, Z, 0, 64, P, P, 4, 64), 6, "null"),
    ("mxfp4_quantize_stream", (Z, P, 0, 64, ODD, P, 4, 64), 6, "aligned"),
    ("mxfp4_dequantize_stream", (Z, P, P, Z, 0, 4, 64), 6, "null"),
    ("mxfp4_linear_stream", (Z, P, 0, 64, P, P, Z, 0, P, 40, 8, 64, Z, 0), 6, "work"),
    ("mxfp4_linear_stream", (Z, P, 0, 64, P, P, Z, 0, P, 40, 8, 64, P, 64), 2, "workspace_size"),
    ("mxfp4_linear_stream", (Z, P, 0, 64, P, P, P, 5, P, 4, 8, 64, Z, 0), 6, "bias_type"),
    ("mxfp4_linear_stream", (Z, P, 0, 64, P, P, Z, 0, P, 4, 0, 64, Z, 0), 2, "positive"),
    ("mxfp4_linear_stream", (Z, P, 0, 64, P, P, Z, 0, P, 1 << 31, 8, 64, Z, 0), 4, "2^31"),
    ("mxfp4_linear_stream", (Z, P, 0, 1 << 20, P, P, Z, 0, P, 1 << 20, 8, 1 << 20, Z, 0), 4, "2^32"),
    ("mxfp4_grouped_linear_stream", (Z, P, 0, 64, P, 4, P, P, Z, 4, P, 8, 8, 64, Z, 0), 6, "offsets"),
    ("mxfp4_grouped_linear_stream", (Z, P, 0, 64, P, 4, P, P, P, 1025, P, 8, 8, 64, Z, 0), 2, "1024"),
    ("mxfp4_grouped_linear_stream", (Z, P, 0, 64, Z, 4, P, P, P, 4, P, 8, 8, 64, Z, 0), 2, "R rows"),
    ("mxfp4_dx_stream", (Z, P, 0, 8, P, P, Z, 0, P, 0, 4, 9, 64, Z, 0), 2, "stride"),
    ("mxfp4_dx_stream", (Z, P, 2, 8, P, P, Z, 0, P, 0, 4, 8, 64, Z, 0), 6, "work"),
    ("mxfp4_dx_stream", (Z, P, 2, 8, P, P, Z, 0, P, 0, 4, 8, 64, P, 8), 2, "workspace_size"),
    ("mxfp4_dx_stream", (Z, P, 0, 8, P, P, Z, 0, P, 7, 4, 8, 64, P, 8), 6, "dx_type"),
    ("moe_sort_stream", (Z, P, 2, P, P, P, P, 4, 2, 4, Z, 0), 2, "ids_int64"),
    ("moe_sort_stream", (Z, P, 0, P, P, P, P, 4, 2, 0, Z, 0), 2, "experts"),
    ("moe_sort_stream", (Z, P, 0, P, Z, P, P, 4, 2, 4, Z, 0), 6, "null"),
    ("moe_sort_stream", (Z, P, 0, P, P, P, P, 40000, 2, 4, Z, 0), 6, "work"),
    ("moe_sort_stream", (Z, P, 0, P, P, P, P, 1 << 30, 2, 4, Z, 0), 4, "2^31"),
    ("moe_dispatch_stream", (Z, P, 0, 8, P, P, P, 4, 2, 4, 9), 2, "stride"),
    ("moe_combine_stream", (Z, P, 0, 8, P, P, P, P, 1, 4, 2, 4, 8), 6, "out_type"),
    ("moe_combine_stream", (Z, P, 0, 8, P, P, P, P, 0, 4, 2, 4, 0), 2, "positive"),
    ("moe_combine_grad_stream", (Z, P, 0, 8, P, 8, P, P, Z, P, P, 4, 2, 4, 8), 6, "weights"),
])
def test_library_refusals(lib, fn, args, code, substr):
    rc = getattr(lib, "xpuint8_" + fn)(*args)
    msg = lib.xpuint8_last_error().decode()
    assert rc == code and substr in msg, (rc, msg)


def test_library_sizes(lib):
    assert lib.xpuint8_mxfp4_scale_width(1280) == 48 and lib.xpuint8_mxfp4_scale_width(48) == -1
    assert lib.xpuint8_mxfp4_linear_workspace_size(4, 8, 48) == -1
    assert lib.xpuint8_mxfp4_linear_workspace_size(100, 8, 1 << 24) > 0
    assert lib.xpuint8_mxfp4_linear_workspace_size(100, 8, (1 << 24) + 32) == -1
    assert b"2^24" in lib.xpuint8_last_error()
    assert lib.xpuint8_mxfp4_dx_workspace_size(0, 0, 100, 0, 8, (1 << 24) + 32) == -1
    assert lib.xpuint8_mxfp4_linear_workspace_size(1000, 8, 64) >= 1000 * (32 + 16)
    assert lib.xpuint8_mxfp4_grouped_linear_workspace_size(8, 4, 0, 8, 64) == -1
    assert lib.xpuint8_mxfp4_dx_workspace_size(2, 2, 10, 0, 100, 64) >= 10 * 128 * 3 * 2
    assert lib.xpuint8_mxfp4_dx_workspace_size(0, 0, 10, 0, 100, 48) == -1
    assert lib.xpuint8_moe_sort_workspace_size(4, 2, 4) == 0


def test_oracle_quantizer_examples():
    """The oracle against values worked out by hand."""
    x = torch.zeros(1, 32)
    x[0, :10] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -7.9, -0.0])
    codes, scales = O.quantize(x)
    v = O.dequantize(codes, scales)[0, :10]
    assert v.tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -6, 0] and scales[0, 0] == 127
    assert torch.signbit(v[9])
    assert O.quantize(x * 0.5)[1][0, 0] == 126 and O.quantize(x * 0)[1][0, 0] == 0
    assert O.quantize(torch.full((1, 32), 2.0 ** 127))[1][0, 0] == 127 + 125
