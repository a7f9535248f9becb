"""Refusals and sizes of the MXFP4 and mixture-of-experts entries beyond those of
test_mx_contract, without a device."""

import ctypes

import pytest

from xpu_kernels.int8 import _lib as L

P, Z, ODD = ctypes.c_void_p(0x1000), ctypes.c_void_p(0), ctypes.c_void_p(0x1008)


@pytest.fixture(scope="module")
def lib():
    path = L.library_path()
    assert path is not None, "libxpuint8.so is not built (run __graft_entry__.build())"
    return L.open_library(path)


@pytest.mark.parametrize("fn,args,code,substr", [
    # stream, dy, type, ldy, dbias, dbias_type, M, N, work, work_bytes
    ("mxfp4_dbias_stream", (Z, P, 0, 8, P, 0, 0, 8, P, 32), 2, "positive"),
    ("mxfp4_dbias_stream", (Z, P, 0, 8, P, 0, 1 << 31, 8, P, 32), 4, "2^31"),
    ("mxfp4_dbias_stream", (Z, P, 0, 1 << 28, P, 0, 1, 1 << 28, P, 32), 4, "2^28"),
    ("mxfp4_dbias_stream", (Z, P, 3, 8, P, 0, 4, 8, P, 32), 6, "type"),
    ("mxfp4_dbias_stream", (Z, P, 0, 8, P, 3, 4, 8, P, 32), 6, "dbias_type"),
    ("mxfp4_dbias_stream", (Z, P, 0, 7, P, 0, 4, 8, P, 32), 2, "stride"),
    ("mxfp4_dbias_stream", (Z, Z, 0, 8, P, 0, 4, 8, P, 32), 6, "null"),
    ("mxfp4_dbias_stream", (Z, P, 0, 8, ODD, 0, 4, 8, P, 32), 6, "aligned"),
    ("mxfp4_dbias_stream", (Z, P, 0, 8, P, 0, 4, 8, Z, 32), 6, "work"),
    ("mxfp4_dbias_stream", (Z, P, 0, 8, P, 0, 33, 8, P, 63), 2, "workspace_size"),
])
def test_library_refusals(lib, fn, args, code, substr):
    rc = getattr(lib, "xpuint8_" + fn)(*args)
    msg = lib.xpuint8_last_error().decode()
    assert rc == code and substr in msg, (rc, msg)


def test_bias_gradient_workspace(lib):
    """One fp32 sum a column (whole 8s of them) and 32 rows."""
    size = lib.xpuint8_mxfp4_dbias_workspace_size
    assert size(1, 1) == size(32, 8) == 32 and size(33, 9) == 2 * 64
    assert size(0, 8) == size(8, 0) == size(1, 1 << 28) == -1


def test_dx_workspace_of_a_dy(lib):
    """What dx takes beside its result: nothing where dy is read where it lies, its bf16
    pieces where it is not, the weight as bf16 where dx goes through it."""
    of, any_dy = lib.xpuint8_mxfp4_dx_workspace_size_of, lib.xpuint8_mxfp4_dx_workspace_size
    # experts: dy, type, ldy, dx_type, R, E, N, K
    assert of(P, 0, 4096, 2, 1000, 8, 4096, 256) == 0
    assert of(P, 0, 8192, 0, 1000, 8, 4096, 256) == 0
    pieces = 1000 * 4096 * 2
    assert of(ODD, 0, 4096, 0, 1000, 8, 4096, 256) == any_dy(0, 0, 1000, 8, 4096, 256) == pieces
    assert of(P, 0, 4100, 0, 1000, 8, 4096, 256) == pieces
    assert of(P, 1, 4096, 1, 1000, 8, 4096, 256) == 2 * pieces
    assert of(P, 2, 4096, 2, 1000, 8, 4096, 256) == 3 * pieces
    # one weight, by tiles and through its bf16 values
    assert of(P, 0, 2048, 0, 64, 0, 2048, 8192) == 0
    through = of(P, 0, 5120, 0, 4096, 0, 5120, 1280)
    assert through >= 2 * 5120 * 1280
    assert any_dy(0, 0, 4096, 0, 5120, 1280) >= max(through, 4096 * 5120 * 2)
    assert of(P, 0, 5128, 0, 4096, 0, 5120, 1280) == 0
    assert of(P, 0, 64, 0, 4, 0, 64, 48) == of(P, 3, 64, 0, 4, 0, 64, 64) == -1


@pytest.mark.parametrize("args,code,substr", [
    # stream, dy, type, ldy, codes, scales, offsets, E, dx, dx_type, R, N, K, work, work_bytes
    ((Z, P, 0, 5120, P, P, Z, 0, P, 0, 4096, 5120, 1280, Z, 0), 6, "work"),
    ((Z, P, 0, 5120, P, P, Z, 0, P, 0, 4096, 5120, 1280, P, 64), 2, "workspace_size"),
    ((Z, ODD, 0, 4096, P, P, P, 8, P, 0, 1000, 4096, 256, P, 1000 * 4096 * 2 - 1), 2, "workspace_size"),
])
def test_dx_refuses_too_little_work(lib, args, code, substr):
    rc = lib.xpuint8_mxfp4_dx_stream(*args)
    msg = lib.xpuint8_last_error().decode()
    assert rc == code and substr in msg, (rc, msg)


def test_products_of_more_blocks_than_a_launch_has(lib):
    """Refused by the sizes already, before anything is allocated."""
    tile, few = (1024 * 65, 1024, 1024, 1 << 22, 32), (1024, 1024, 1024, 1 << 22, 32)
    assert lib.xpuint8_mxfp4_grouped_linear_workspace_size(*tile) == -1
    assert b"one launch" in lib.xpuint8_last_error()
    assert lib.xpuint8_mxfp4_grouped_linear_workspace_size(*few) == 0
    assert lib.xpuint8_mxfp4_dx_workspace_size(0, 0, 1024, 1024, 8, 1 << 24) == -1
    assert b"one launch" in lib.xpuint8_last_error()
    assert lib.xpuint8_mxfp4_dx_workspace_size(0, 0, 1024, 1, 8, 1 << 24) > 0
    # 48 GiB of bf16 results are not too many
    assert lib.xpuint8_mxfp4_linear_workspace_size(1 << 20, 24576, 4096) > 0
    assert lib.xpuint8_mxfp4_dx_workspace_size(0, 0, 1 << 20, 0, 4096, 24576) > 0


@pytest.mark.parametrize("fn,args,code,substr", [
    ("mxfp4_grouped_linear_stream", (Z, P, 0, 32, P, 1024, P, P, P, 1024, P, 66560, 1 << 22, 32, P, 1 << 40),
     4, "one launch"),
    ("mxfp4_dx_stream", (Z, P, 0, 8, P, P, P, 1024, P, 0, 1024, 8, 1 << 24, Z, 0), 4, "one launch"),
    ("moe_dispatch_stream", (Z, P, 0, 8, P, P, P, 1 << 31, 1, 4, 8), 4, "2^31"),
    ("moe_combine_stream", (Z, P, 0, 8, P, P, P, P, 0, 4, 2, 1025, 8), 2, "1024"),
])
def test_refusals_of_sizes(lib, fn, args, code, substr):
    rc = getattr(lib, "xpuint8_" + fn)(*args)
    msg = lib.xpuint8_last_error().decode()
    assert rc == code and substr in msg, (rc, msg)
