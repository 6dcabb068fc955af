"""What the gated delta rule refuses before anything is launched, and its workspace: no device needed."""
import ctypes as C
import importlib

import pytest

fr = importlib.import_module("faster-rwkv_amd")
EINVAL, ESHAPE = -1, -2
A = 1 << 22  # addresses that nothing reads


def starts(*v):
    return (C.c_int32 * len(v))(*v)


def params(**kw):
    p = dict(A=A, bias=2 * A, heads=4, key_heads=2, dk=32, dv=16, scale=1.0, eps=1e-6, softplus=1, sigmoid=1)
    p.update(kw)
    return C.byref(fr.Delta(*p.values()))


def delta(seq=True, p=None, **kw):
    v = dict(n=1, at=starts(0, 4), q=3 * A, ldq=64, k=4 * A, ldk=64, v=5 * A, ldv=64, dt=6 * A, lddt=4, beta=7 * A, ldbeta=4, state=8 * A, out=9 * A,
             y=10 * A, ldy=64, dtype=fr.F16, ws=11 * A)
    v.update(kw)
    mid = [v[k] for k in ("q", "ldq", "k", "ldk", "v", "ldv", "dt", "lddt", "beta", "ldbeta", "state", "out", "y", "ldy", "dtype")]
    if seq:
        return fr.lib().frhip_delta_seq(params(**(p or {})), v["n"], v["at"], *mid, v["ws"], None)
    return fr.lib().frhip_delta_one(params(**(p or {})), v["n"], *mid, None)


@pytest.mark.parametrize("seq", [True, False])
@pytest.mark.parametrize("kw,code", [
    (dict(n=-1), ESHAPE), (dict(ldq=63), ESHAPE), (dict(ldq=(1 << 23) + 1), ESHAPE), (dict(ldy=(1 << 23) + 1), ESHAPE), (dict(ldk=63), ESHAPE), (dict(ldv=63), ESHAPE), (dict(lddt=3), ESHAPE), (dict(ldbeta=3), ESHAPE),
    (dict(ldy=63), ESHAPE), (dict(q=None), EINVAL), (dict(k=None), EINVAL), (dict(v=None), EINVAL), (dict(dt=None), EINVAL), (dict(beta=None), EINVAL),
    (dict(state=None), EINVAL), (dict(out=None), EINVAL), (dict(y=None), EINVAL), (dict(dtype=fr.U8), EINVAL), (dict(q=3 * A + 1), EINVAL), (dict(state=8 * A + 2), EINVAL),
    (dict(y=3 * A), EINVAL), (dict(y=4 * A + 2), EINVAL), (dict(y=5 * A), EINVAL), (dict(y=6 * A), EINVAL), (dict(y=7 * A + 2), EINVAL), (dict(y=8 * A), EINVAL),
    (dict(y=9 * A + 64), EINVAL), (dict(out=8 * A + 4), EINVAL), (dict(out=5 * A), EINVAL), (dict(p=dict(A=10 * A)), EINVAL), (dict(p=dict(bias=9 * A)), EINVAL),
    (dict(p=dict(A=A + 2)), EINVAL), (dict(p=dict(heads=3)), ESHAPE), (dict(p=dict(heads=0)), ESHAPE), (dict(p=dict(key_heads=0)), ESHAPE), (dict(p=dict(dk=0)), ESHAPE),
    (dict(p=dict(heads=65536, key_heads=1, dv=1), lddt=65536, ldbeta=65536, ldv=65536, ldy=65536), ESHAPE), (dict(p=dict(dk=257)), ESHAPE), (dict(p=dict(dv=0)), ESHAPE), (dict(p=dict(dv=257)), ESHAPE), (dict(p=dict(heads=1 << 22, key_heads=1), ldv=1 << 27, ldy=1 << 27), ESHAPE)])
def test_refusals(kw, code, seq):
    assert delta(seq, **kw) == code and fr.lib().frhip_error_string()


def test_starts_and_row_numbers():
    assert delta(at=None) == EINVAL
    assert delta(at=starts(-1, 4)) == delta(n=2, at=starts(0, 4, 3)) == delta(at=starts(0, (1 << 28) + 1)) == ESHAPE
    assert delta(False, n=(1 << 30) + 1) == ESHAPE


def test_no_struct():
    v = [A, 64, A, 64, A, 64, A, 4, A, 4, A, 2 * A, 3 * A, 64, 1]
    assert fr.lib().frhip_delta_one(None, 1, *v, None) == EINVAL and fr.lib().frhip_delta_seq(None, 1, starts(0, 1), *v, None, None) == EINVAL
    assert fr.lib().frhip_delta_workspace_bytes(None, 1, 100) == 0


def test_nothing_to_do():
    assert delta(n=0, at=None) == 0 and delta(False, n=0) == 0


@pytest.mark.parametrize("heads,key_heads,dk,dv", [(1, 1, 1, 1), (4, 2, 32, 16), (24, 24, 64, 64), (32, 16, 128, 128), (6, 3, 256, 256), (3, 1, 17, 203)])
def test_a_workspace_for_more_rows_serves_fewer(heads, key_heads, dk, dv):
    p = params(heads=heads, key_heads=key_heads, dk=dk, dv=dv)
    sizes = [fr.lib().frhip_delta_workspace_bytes(p, n, T) for T in [*range(600), 4096, 100000, 1 << 28] for n in (1, 200)]
    assert sizes == sorted(sizes) and sizes[0::2] == sizes[1::2]


@pytest.mark.parametrize("seq", [True, False])
@pytest.mark.parametrize("eps", [float("nan"), float("inf")])
def test_an_eps_that_is_no_number(eps, seq):
    assert delta(seq, p=dict(eps=eps)) == EINVAL


def test_a_workspace_that_is_not_there_or_off_its_grid():
    for ws in (None, 11 * A + 8):
        assert delta(at=starts(0, 100), ws=ws, q=3 * A, k=13 * A) == EINVAL
