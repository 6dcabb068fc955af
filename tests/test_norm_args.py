"""What the fused norms refuse before anything is launched: no device needed."""
import ctypes as C
import importlib

import pytest

fr = importlib.import_module("faster-rwkv_amd")
EINVAL, ESHAPE = -1, -2
A = 1 << 20  # addresses that nothing reads
NAN = float("nan")


def gate(**kw):
    v = dict(rows=4, heads=2, dim=32, kind=1, w=A, b=2 * A, eps=1e-6, x=3 * A, ldx=64, z=4 * A, ldz=64, act=4, y=5 * A, ldy=64, dtype=fr.F16)
    v.update(kw)
    return fr.lib().frhip_norm_gate(*v.values(), None)


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), ESHAPE), (dict(rows=(1 << 30) + 1), ESHAPE), (dict(heads=0), ESHAPE), (dict(dim=0), ESHAPE), (dict(dim=(1 << 15) + 1, heads=1, ldx=1 << 16, ldz=1 << 16, ldy=1 << 16), ESHAPE),
    (dict(heads=1 << 20, dim=17, ldx=1 << 25, ldz=1 << 25, ldy=1 << 25), ESHAPE), (dict(kind=0), EINVAL), (dict(kind=3), EINVAL), (dict(act=3), EINVAL), (dict(act=6), EINVAL),
    (dict(eps=-1e-6), EINVAL), (dict(eps=NAN), EINVAL), (dict(dtype=fr.U8), EINVAL), (dict(ldx=63), ESHAPE), (dict(ldz=63), ESHAPE), (dict(ldy=63), ESHAPE),
    (dict(x=None), EINVAL), (dict(y=None), EINVAL), (dict(x=3 * A + 1), EINVAL), (dict(w=A + 2), EINVAL), (dict(dtype=fr.F32, z=4 * A + 2), EINVAL),
    (dict(y=3 * A + 2), EINVAL), (dict(y=3 * A, ldy=65), EINVAL), (dict(y=4 * A), EINVAL), (dict(w=5 * A + 4), EINVAL), (dict(b=5 * A), EINVAL)])
def test_gate_refusals(kw, code):
    assert gate(**kw) == code and fr.lib().frhip_error_string()


def residual(params=None, **kw):
    p = dict(aw=A, ab=2 * A, bw=3 * A, bb=4 * A, channels=5 * A, cols=64, after=1, before=2, act=2, scale=1.0, eps=1e-6)
    p.update(params or {})
    v = dict(rows=4, x=6 * A, ldx=64, block=7 * A, ldb=64, gate=8 * A, ldg=64, h=9 * A, ldh=64, sdtype=fr.F32, y=10 * A, ldy=64, dtype=fr.F16)
    v.update(kw)
    return fr.lib().frhip_norm_residual(C.byref(fr.BlockNorm(*p.values())), *v.values(), None)


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), ESHAPE), (dict(rows=(1 << 30) + 1), ESHAPE), (dict(params=dict(cols=0)), ESHAPE),
    (dict(params=dict(cols=(1 << 15) + 1), ldx=1 << 16, ldb=1 << 16, ldg=1 << 16, ldh=1 << 16, ldy=1 << 16), ESHAPE), (dict(params=dict(after=3)), EINVAL),
    (dict(params=dict(before=-1)), EINVAL), (dict(params=dict(act=5)), EINVAL), (dict(params=dict(eps=-1.0)), EINVAL), (dict(params=dict(eps=NAN)), EINVAL),
    (dict(sdtype=fr.U8), EINVAL), (dict(dtype=7), EINVAL), (dict(ldx=63), ESHAPE), (dict(ldb=63), ESHAPE), (dict(ldg=63), ESHAPE), (dict(ldg=-1), ESHAPE), (dict(ldh=63), ESHAPE),
    (dict(ldy=63), ESHAPE), (dict(x=None), EINVAL), (dict(h=None, y=None), EINVAL), (dict(block=None), EINVAL), (dict(x=6 * A + 2), EINVAL), (dict(block=7 * A + 1), EINVAL),
    (dict(params=dict(channels=5 * A + 1)), EINVAL), (dict(h=6 * A + 4), EINVAL), (dict(h=6 * A, ldh=65), EINVAL), (dict(h=7 * A), EINVAL), (dict(y=7 * A), EINVAL),
    (dict(y=8 * A), EINVAL), (dict(y=8 * A + 2, ldg=0), EINVAL), (dict(y=6 * A), EINVAL), (dict(y=9 * A), EINVAL), (dict(params=dict(bb=10 * A)), EINVAL),
    (dict(params=dict(aw=9 * A + 8)), EINVAL)])
def test_residual_refusals(kw, code):
    assert residual(**kw) == code and fr.lib().frhip_error_string()


def test_no_struct():
    assert fr.lib().frhip_norm_residual(None, 1, A, 8, None, 0, None, 0, 2 * A, 8, 1, None, 0, 1, None) == EINVAL


def test_nothing_to_do():
    assert gate(rows=0) == 0 and residual(rows=0) == 0 and gate(rows=0, x=None, y=None) == 0
