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


ROWS, FEW, TILES, CODES = range(4)


def form(T, K, N, dtype, units=256):
    out = (C.c_int * 3)()
    rc = fr.lib().frhip_linear_form(T, C.byref(fr.Weight(A, A, A, A, A, K, N, dtype)), units, out)
    return rc, tuple(out)


def test_forms():
    """What goes where; uint8 codes that no tile takes as they are, and rows of eight, are expanded"""
    assert form(1, 2048, 2048, fr.F16) == (ROWS, (0, 0, 0)) and form(2, 8, 1, fr.F16)[0] == ROWS
    assert form(3, 2048, 2048, fr.F16)[0] == form(1, 2048, 2048, fr.U8)[0] == FEW
    assert form(1, 8, 2048, fr.U8)[1][2] == 1 and form(1, 16, 2048, fr.U8)[1][2] == form(1, 24, 2048, fr.U8)[1][2] == form(1, 2056, 2048, fr.U8)[1][2] == 0
    assert form(4099, 5120, 2560, fr.F16)[:1] + form(4099, 5120, 2560, fr.F16)[1][:1] == (TILES, 256)
    assert form(512, 2048, 8192, fr.U8)[0] == CODES and form(512, 2056, 8192, fr.U8)[1][2] == form(512, 2048, 8200, fr.U8)[1][2] == 1


def test_rows_behind_whole_tiles_go_out_by_themselves_where_a_strip_of_tiles_costs_a_round():
    assert [form(T, 2048, 8192, fr.F16)[1][2] for T in (2048, 2051)] == [0, 2]
    assert form(1027, 5120, 5120, fr.F16)[1][2] == form(130, 64, 64, fr.F16)[1][2] == 0 and form(1027, 1000, 8192, fr.U8)[1][2] == 3


def test_every_product_has_a_form():
    for units in (1, 64, 256, 304):
        for T in (1, 2, 3, 17, 64, 300, 513, 5000, 1 << 20):
            for K in (8, 56, 64, 1000, 2048, 8388544):
                for N in (1, 17, 2048, 50277, 1 << 20):
                    if K * N > 1 << 34:
                        assert form(T, K, N, fr.F16, units)[0] == ESHAPE
                        continue
                    for dtype in (fr.F16, fr.U8):
                        rc, out = form(T, K, N, dtype, units)
                        assert rc in (ROWS, FEW, TILES, CODES) and (rc == ROWS or out[0] > 0 and out[1] > 0)
                        need = fr.lib().frhip_linear_workspace_bytes(T, C.byref(fr.Weight(A, A, A, A, A, K, N, dtype)))
                        if units == 256:
                            assert (need >= 2 * K * N) == (out[2] & 1 == 1) and (need == 0) == (out[2] & 1 == 0)


def test_form_arguments():
    out = (C.c_int * 3)()
    f, w = fr.lib().frhip_linear_form, C.byref(fr.Weight(A, A, A, A, A, 64, 64, fr.F16))
    assert f(1, None, 256, out) == f(1, w, 256, None) == EINVAL and f(0, w, 256, out) == f(1, w, 0, out) == ESHAPE
    assert form(1, 60, 64, fr.F16)[0] == form(1, 8388552, 64, fr.F16)[0] == form(1, 64, (1 << 24) + 1, fr.F16)[0] == form((1 << 30) + 1, 64, 64, fr.F16)[0] == ESHAPE


@pytest.mark.parametrize("K,N", [(2048, 8192), (4096, 2048), (5120, 2048), (64, 8192), (128, 2048), (512, 10240), (4096, 50288), (2048, 512), (64, 1 << 20),
                                 (8, 40), (24, 8192), (2056, 8192), (2048, 8200), (64, 160)])
def test_a_workspace_for_some_rows_serves_fewer(K, N):
    """Codes are expanded at some numbers of rows and not at others above them: what one call writes, a workspace for more rows holds"""
    w, most = fr.Weight(A, A, A, A, A, K, N, fr.U8), 0
    for T in range(1, 2400):
        if form(T, K, N, fr.U8)[1][2] & 1:
            most = 2 * K * N
        if T % 64 in (0, 1, 33) or T < 140:
            assert fr.lib().frhip_linear_workspace_bytes(T, C.byref(w)) >= most, T
    sizes = [fr.lib().frhip_linear_workspace_bytes(T, C.byref(w)) for T in (1, 16, 100, 512, 513, 1024, 1153, 1409, 3000, 4100, 8192, 8193, 100000, 1 << 30)]
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("kw", [dict(y=A + 124, ldy=64), dict(y=A + 132, ldy=64), dict(y=A + 252, ldy=64), dict(y=A + 128, ldy=66)])
def test_rows_of_fp32_beside_those_of_x_that_overlap_them(kw):
    """x: 64 of 128 binary16 a row of 256 bytes; y: 32 fp32 at a byte of such a row"""
    assert linear(ldx=128, out=fr.F32, **kw) == EINVAL
