"""The fused norms at the ends of what they take: the largest and smallest values whose squares and their sums are fp32 numbers, in the longest rows."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from hipref import DevBuf, L, dev, fr
from test_gpu_norm import NORM, close, norm64

ROWS = 3


def values(dim, size, lone):
    """Row by row: all elements at the limit, half of them, and (lone) one alone beside zeros"""
    g = np.random.default_rng(dim)
    x = g.choice([-1.0, 1.0], (ROWS, dim)) * size
    x[1, ::2] *= g.uniform(0, 1, x[1, ::2].shape)
    if lone:
        x[2] = 0
        x[2, dim // 2] = size
    return x.astype(np.float32)


@pytest.mark.parametrize("kind", ["rms", "mean"])
@pytest.mark.parametrize("dim", [64, 600, 32768])
@pytest.mark.parametrize("size,lone,eps", [(0.9999e17, False, 1e-6), (0.9999e17, True, 0.0), (1.001e-16, True, 0.0), (1.001e-16, False, 0.0)])
def test_gate_and_residual(size, lone, eps, dim, kind):
    x = values(dim, size, lone)
    v = x.astype(np.float64)
    want, err = norm64(v, np.zeros_like(v), kind, None, None, eps)
    dx, y, h = dev(x), DevBuf.empty(x.shape, np.float32), DevBuf.empty(x.shape, np.float32)
    fr.check(L().frhip_norm_gate(ROWS, 1, dim, NORM[kind], None, None, eps, dx.ptr, dim, None, 0, 0, y.ptr, dim, fr.F32, None), "norm_gate")
    fr.check(L().frhip_device_sync())
    close(y.numpy(), want, err, np.float32)
    # of the stream itself, and of a block that the stream (zeros) is added to
    p = fr.BlockNorm(None, None, None, None, None, dim, 0, NORM[kind], 0, 1.0, eps)
    fr.check(L().frhip_norm_residual(C.byref(p), ROWS, dx.ptr, dim, None, 0, None, 0, None, 0, fr.F32, y.ptr, dim, fr.F32, None), "norm_residual")
    fr.check(L().frhip_device_sync())
    close(y.numpy(), want, err, np.float32)
    zeros = dev(np.zeros_like(x))
    p = fr.BlockNorm(None, None, None, None, None, dim, NORM[kind], 0, 0, 1.0, eps)
    fr.check(L().frhip_norm_residual(C.byref(p), ROWS, zeros.ptr, dim, dx.ptr, dim, None, 0, h.ptr, dim, fr.F32, None, 0, fr.F32, None), "norm_residual")
    fr.check(L().frhip_device_sync())
    close(h.numpy(), want, err, np.float32)
