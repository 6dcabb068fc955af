"""The fused norms over more rows than their workgroups take at once, so that each goes on to further rows, and over the largest and smallest values."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from hipref import L, dev, fr
from test_gpu_norm import EPS, close, gate_case, norm64, residual_case


def compute_units():
    n = C.c_int()
    fr.check(L().frhip_device_info(None, 0, C.byref(n), None))
    return n.value


# A launch has workgroups of `threads` threads for 4096 (residual) or 2048 (gate) of them a compute unit at most
def rows_of_a_pass(total, cols, at_once=1):
    threads = min(1024, (-(-cols // 8) + 63) // 64 * 64)
    return compute_units() * (total // threads) * at_once


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("stream,dtype", [("f16", "f16"), ("f32", "f16"), ("f32", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("kw", [dict(), dict(after="rms"), dict(after="mean", gate="silu"), dict(after="rms", before="mean", channels=True),
                                dict(after="mean", before="mean")])
def test_residual_of_short_rows(kw, stream, dtype, in_place):
    """One to four sums a row; a wave a row, four rows a workgroup"""
    residual_case(2 * compute_units() * 16 * 4 + 77, 40, stream=stream, dtype=dtype, in_place=in_place, **kw)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("stream,dtype", [("f16", "f16"), ("f32", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("cols,kw", [(600, dict()), (600, dict(after="rms")), (601, dict(after="mean", gate="sigmoid")), (600, dict(after="mean", before="mean", channels=True)),
                                     (2560, dict(after="rms", gate="silu")), (1545, dict(before="mean")), (8200, dict(after="rms", before="mean")), (8200, dict()),
                                     (16400, dict(after="rms", gate="sigmoid")), (16393, dict(before="mean"))])
def test_residual_of_rows_of_a_workgroup(cols, kw, stream, dtype, in_place):
    """One to four sums a row, odd and even; two rows and a little more a workgroup"""
    residual_case(2 * rows_of_a_pass(4096, cols) + 5, cols, stream=stream, dtype=dtype, in_place=in_place, **kw)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("kind", ["rms", "mean"])
@pytest.mark.parametrize("heads,dim", [(1, 600), (2, 600), (1, 1545), (1, 5000), (1, 8200), (1, 20000)])
def test_gate_of_rows_of_a_workgroup(heads, dim, kind, dtype):
    close(*gate_case(2 * rows_of_a_pass(2048, dim) // heads + 5, heads, dim, kind, dtype=dtype, b=kind == "mean", in_place=dtype == "f32"))


@pytest.mark.parametrize("heads,dim", [(1, 8), (3, 64), (5, 130), (2, 300)])
def test_gate_of_rows_of_lanes(heads, dim):
    """As many rows as two passes of 32 waves a compute unit have"""
    lanes = 8 if dim <= 64 else 16 if dim <= 128 else 32 if dim <= 256 else 64
    close(*gate_case(2 * compute_units() * 2048 // lanes // heads + 77, heads, dim, "mean", b=True))
