"""What frhip_linear refuses before anything is launched: no device needed."""
import ctypes as C
import importlib

import pytest

fr = importlib.import_module("faster-rwkv_amd")
EINVAL, ESHAPE = -1, -2
A = 1 << 20  # addresses that nothing reads


def linear(weight=None, **kw):
    w = dict(data=2 * A, mx=None, rx=None, my=None, ry=None, K=64, N=32, dtype=fr.F16)
    w.update(weight or {})
    v = dict(x=A, ldx=64, bias=None, act=0, res=None, ldr=32, y=3 * A, ldy=32, T=4, out=fr.F16, ws=None)
    v.update(kw)
    return fr.lib().frhip_linear(v["x"], v["ldx"], C.byref(fr.Weight(*w.values())), v["bias"], v["act"], v["res"], v["ldr"], v["y"], v["ldy"], v["T"],
                                 v["out"], v["ws"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), EINVAL), (dict(y=None), EINVAL), (dict(T=-1), ESHAPE), (dict(ldx=56), ESHAPE), (dict(ldx=68), ESHAPE), (dict(ldy=31), ESHAPE),
    (dict(res=4 * A, ldr=31), ESHAPE), (dict(act=1), EINVAL), (dict(act=7), EINVAL), (dict(act=-1), EINVAL), (dict(out=fr.U8), EINVAL), (dict(x=A + 8), EINVAL),
    (dict(y=3 * A + 1), EINVAL), (dict(y=3 * A + 2, out=fr.F32), EINVAL), (dict(bias=A + 2), EINVAL), (dict(res=4 * A + 1), EINVAL), (dict(y=A), EINVAL),
    (dict(y=A + 64 * 6, ldy=64), EINVAL), (dict(y=2 * A), EINVAL), (dict(res=3 * A + 2), EINVAL), (dict(res=3 * A, ldr=33), EINVAL), (dict(bias=3 * A), EINVAL),
    (dict(weight=dict(K=60)), ESHAPE), (dict(weight=dict(K=0)), ESHAPE), (dict(weight=dict(N=0)), ESHAPE), (dict(weight=dict(data=None)), EINVAL),
    (dict(weight=dict(data=2 * A + 8)), EINVAL), (dict(weight=dict(dtype=fr.F32)), EINVAL), (dict(weight=dict(dtype=fr.U8)), EINVAL),
    (dict(weight=dict(dtype=fr.U8, mx=A, rx=A, my=A, ry=A + 1)), EINVAL)])
def test_refusals(kw, code):
    assert linear(**kw) == code and fr.lib().frhip_error_string()


def test_no_weight_and_no_rows():
    f = fr.lib().frhip_linear
    assert f(A, 64, None, None, 0, None, 0, 3 * A, 32, 4, fr.F16, None, None) == EINVAL
    assert linear(T=0, x=None, y=None) == 0
    assert fr.lib().frhip_linear_workspace_bytes(4, None) == 0
