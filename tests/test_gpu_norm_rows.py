"""The fused norms over more rows than their workgroups take at once, so that each goes on to further rows, and over the largest and smallest values."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

from hipref import L, fr
from test_gpu_norm import close, gate_case, residual_case


def compute_units():
    n = C.c_int()
    fr.check(L().frhip_device_info(None, 0, C.byref(n), None))
    return n.value


# A launch has workgroups of `threads` threads for 4096 (residual) or 2048 (gate) of them a compute unit at most
def rows_of_a_pass(total, cols):
    threads = min(1024, (-(-cols // 8) + 63) // 64 * 64)
    return compute_units() * (total // threads)


@pytest.mark.parametrize("in_place,stream,dtype", [(True, "f16", "f16"), (False, "f32", "f16"), (True, "f32", "f32")])
@pytest.mark.parametrize("kw", [dict(), dict(after="rms"), dict(after="mean", gate="silu"), dict(after="mean", before="mean", channels=True)])
def test_residual_of_short_rows(kw, stream, dtype, in_place):
    """One to four sums a row; a wave a row, four rows a workgroup; two passes and a little more"""
    residual_case(2 * compute_units() * 16 * 4 + 77, 40, stream=stream, dtype=dtype, in_place=in_place, **kw)


@pytest.mark.parametrize("cols,stream,dtype,in_place,kw", [
    (600, "f16", "f16", False, dict()), (600, "f32", "f16", True, dict(after="rms")), (601, "f16", "f16", True, dict(after="mean", gate="sigmoid")),
    (600, "f32", "f32", True, dict(after="mean", before="mean", channels=True)), (1545, "f16", "f32", True, dict(before="mean")),
    (2560, "f32", "f16", True, dict(after="rms", gate="silu")), (8200, "f16", "f16", True, dict(after="rms", before="mean")), (8200, "f32", "f32", False, dict()),
    (16400, "f16", "f16", True, dict(after="rms", gate="sigmoid")), (16393, "f32", "f16", True, dict(before="mean"))])
def test_residual_of_rows_of_a_workgroup(cols, stream, dtype, in_place, kw):
    """One to four sums a row, odd and even; a pass and a half, a little more than two of rows of 600"""
    rows = rows_of_a_pass(4096, cols)
    residual_case(rows * 2 + 5 if cols <= 601 else rows * 3 // 2, cols, stream=stream, dtype=dtype, in_place=in_place, **kw)


@pytest.mark.parametrize("heads,dim,kind,dtype", [(1, 600, "rms", "f16"), (1, 600, "mean", "f32"), (2, 600, "mean", "f16"), (1, 1545, "rms", "f32"), (1, 5000, "mean", "f16"),
                                                  (1, 8200, "rms", "f32"), (1, 20000, "mean", "f16")])
def test_gate_of_rows_of_a_workgroup(heads, dim, kind, dtype):
    close(*gate_case(rows_of_a_pass(2048, dim) // heads * 3 // 2 + 5, heads, dim, kind, dtype=dtype, b=kind == "mean", in_place=dtype == "f32"))


@pytest.mark.parametrize("heads,dim", [(1, 8), (3, 64), (5, 130), (2, 300)])
def test_gate_of_rows_of_lanes(heads, dim):
    """As many rows as two passes of 32 waves a compute unit have"""
    lanes = 8 if dim <= 64 else 16 if dim <= 128 else 32 if dim <= 256 else 64
    close(*gate_case(2 * compute_units() * 2048 // lanes // heads + 77, heads, dim, "mean", b=True))
