"""What the state space operators refuse before anything is launched, and how the scan is cut: no device needed."""
import ctypes as C
import importlib

import pytest

fr = importlib.import_module("faster-rwkv_amd")
EINVAL, ESHAPE = -1, -2
A = 1 << 20  # addresses that nothing reads


def starts(*v):
    return (C.c_int32 * len(v))(*v)


def conv(seq=True, **kw):
    v = dict(n=1, at=starts(0, 4), C=8, W=4, x=A, ldx=8, w=2 * A, bias=None, act=4, state=3 * A, out=4 * A, y=5 * A, ldy=8, dtype=fr.F16)
    v.update(kw)
    tail = [v[k] for k in ("C", "W", "x", "ldx", "w", "bias", "act", "state", "out", "y", "ldy", "dtype")] + [None]
    return fr.lib().frhip_conv_seq(v["n"], v["at"], *tail) if seq else fr.lib().frhip_conv_one(v["n"], *tail)


@pytest.mark.parametrize("seq", [True, False])
@pytest.mark.parametrize("kw,code", [
    (dict(n=-1), ESHAPE), (dict(C=0), ESHAPE), (dict(W=1), ESHAPE), (dict(W=5), ESHAPE), (dict(ldx=7), ESHAPE), (dict(ldy=7), ESHAPE),
    (dict(x=None), EINVAL), (dict(w=None), EINVAL), (dict(state=None), EINVAL), (dict(out=None), EINVAL), (dict(y=None), EINVAL),
    (dict(act=2), EINVAL), (dict(dtype=fr.U8), EINVAL), (dict(x=A + 1), EINVAL), (dict(w=2 * A + 2), EINVAL), (dict(dtype=fr.F32, y=5 * A + 2), EINVAL),
    (dict(y=A), EINVAL), (dict(y=A + 14), EINVAL), (dict(out=3 * A + 2), EINVAL), (dict(y=3 * A), EINVAL), (dict(y=4 * A + 40), EINVAL), (dict(out=A), EINVAL),
    (dict(w=5 * A + 4), EINVAL), (dict(bias=5 * A), EINVAL), (dict(w=4 * A), EINVAL)])
def test_conv_refusals(kw, code, seq):
    assert conv(seq, **kw) == code and fr.lib().frhip_error_string()


def test_conv_seq_refuses_starts_that_descend():
    assert conv(at=None) == EINVAL
    assert conv(at=starts(-1, 4)) == ESHAPE and conv(n=2, at=starts(0, 4, 3)) == ESHAPE


def test_single_tokens_of_too_many_sequences():
    assert conv(False, n=(1 << 30) + 1) == scan(False, n=(1 << 30) + 1) == ESHAPE


def test_row_numbers_and_channels_beyond_the_limits():
    far = starts(0, (1 << 28) + 1)
    assert conv(at=far) == scan(at=far) == ESHAPE
    c = (1 << 24) + 1
    assert conv(C=c, ldx=c, ldy=c) == conv(False, C=c, ldx=c, ldy=c) == ESHAPE
    for seq in (True, False):
        assert scan(seq, params=dict(channels=c, groups=1), ldx=c, lddt=c, ldz=c, ldy=c) == ESHAPE


def test_conv_of_nothing():
    assert conv(n=0, at=None) == 0 and conv(False, n=0) == 0


def scan(seq=True, params=None, **kw):
    p = dict(A=A, D=None, bias=None, channels=8, states=4, groups=2, softplus=1)
    p.update(params or {})
    v = dict(n=1, at=starts(0, 4), x=2 * A, ldx=8, dt=3 * A, lddt=8, B=4 * A, ldb=8, C=5 * A, ldc=8, z=6 * A, ldz=8, state=7 * A, out=8 * A,
             y=9 * A, ldy=8, dtype=fr.F16, ws=10 * A)
    v.update(kw)
    ref = C.byref(fr.Ssm(*p.values()))
    mid = [v[k] for k in ("x", "ldx", "dt", "lddt", "B", "ldb", "C", "ldc", "z", "ldz", "state", "out", "y", "ldy", "dtype")]
    if seq:
        return fr.lib().frhip_ssm_seq(ref, v["n"], v["at"], *mid, v["ws"], None)
    return fr.lib().frhip_ssm_one(ref, v["n"], *mid, None)


@pytest.mark.parametrize("seq", [True, False])
@pytest.mark.parametrize("kw,code", [
    (dict(n=-1), ESHAPE), (dict(ldx=7), ESHAPE), (dict(lddt=7), ESHAPE), (dict(ldb=7), ESHAPE), (dict(ldc=7), ESHAPE), (dict(ldz=7), ESHAPE),
    (dict(ldy=7), ESHAPE), (dict(x=None), EINVAL), (dict(dt=None), EINVAL), (dict(B=None), EINVAL), (dict(C=None), EINVAL), (dict(state=None), EINVAL),
    (dict(out=None), EINVAL), (dict(y=None), EINVAL), (dict(dtype=fr.U8), EINVAL), (dict(x=2 * A + 1), EINVAL), (dict(state=7 * A + 2), EINVAL),
    (dict(y=2 * A), EINVAL), (dict(y=6 * A), EINVAL), (dict(y=4 * A + 2), EINVAL), (dict(out=7 * A + 4), EINVAL), (dict(out=2 * A), EINVAL), (dict(y=7 * A), EINVAL),
    (dict(params=dict(A=9 * A)), EINVAL), (dict(params=dict(D=8 * A)), EINVAL), (dict(params=dict(bias=9 * A + 4)), EINVAL), (dict(params=dict(A=None)), EINVAL), (dict(params=dict(A=A + 2)), EINVAL), (dict(params=dict(D=A + 1)), EINVAL), (dict(params=dict(channels=9)), ESHAPE),
    (dict(params=dict(channels=0)), ESHAPE), (dict(params=dict(states=0)), ESHAPE), (dict(params=dict(states=257)), ESHAPE), (dict(params=dict(groups=0)), ESHAPE)])
def test_scan_refusals(kw, code, seq):
    assert scan(seq, **kw) == code and fr.lib().frhip_error_string()


def test_scan_seq_refuses_starts_that_descend_and_a_missing_workspace():
    assert scan(at=None) == EINVAL
    assert scan(at=starts(-1, 4)) == ESHAPE and scan(n=2, at=starts(0, 4, 3)) == ESHAPE
    assert scan(at=starts(0, 400), ws=None) == EINVAL and scan(at=starts(0, 400), ws=10 * A + 8) == EINVAL


def test_scan_of_nothing():
    assert scan(n=0, at=None) == 0 and scan(False, n=0) == 0


@pytest.mark.parametrize("units", [1, 64, 256, 304, 5000])
@pytest.mark.parametrize("channels,states,groups", [(1, 1, 1), (96, 16, 1), (4096, 16, 1), (300, 24, 3), (5120, 256, 1), (100000, 16, 1)])
def test_time_is_covered_and_the_workspace_holds_the_chunks(channels, states, groups, units):
    p = fr.Ssm(A, None, None, channels, states, groups, 1)
    out = (C.c_int * 3)()
    for lens in ([0], [1], [16], [17], [4096], [0, 1, 500, 0, 33], [100000], [2 ** 31 - 1], [7] * 128, [1000] * 128):
        at, total = [0], sum(lens)
        for n in lens:
            at.append(at[-1] + n)
        assert fr.lib().frhip_ssm_cut(C.byref(p), len(lens), starts(*at), units, out) == 0
        rows, chunks, wgs = out
        assert chunks == sum(max(1, -(-n // rows)) for n in lens) <= 65535 and wgs >= 1
        local = chunks - len(lens)
        need = 4 * (2 * local * channels * -(-states // 4) * 4 + local * channels)
        assert need <= fr.lib().frhip_ssm_workspace_bytes(C.byref(p), len(lens), total)


@pytest.mark.parametrize("lens", [[17], [32], [1, 32, 0, 20], [32] * 128])
def test_short_prompts_are_not_cut(lens):
    p, out = fr.Ssm(A, None, None, 64, 16, 1, 1), (C.c_int * 3)()
    at = [sum(lens[:i]) for i in range(len(lens) + 1)]
    assert fr.lib().frhip_ssm_cut(C.byref(p), len(lens), starts(*at), 256, out) == 0 and out[1] == len(lens)


def test_cut_arguments():
    p, out, f = fr.Ssm(A, None, None, 64, 16, 1, 1), (C.c_int * 3)(), fr.lib().frhip_ssm_cut
    assert f(None, 1, starts(0, 4), 256, out) == f(C.byref(p), 1, starts(0, 4), 256, None) == EINVAL
    assert f(C.byref(p), 1, starts(0, 4), 0, out) == f(C.byref(p), 0, None, 256, out) == f(C.byref(p), 129, starts(*range(130)), 256, out) == ESHAPE


@pytest.mark.parametrize("channels,states,groups", [(1, 1, 1), (96, 16, 1), (300, 24, 3), (5120, 256, 1), (100000, 16, 1)])
def test_a_workspace_for_more_rows_serves_fewer(channels, states, groups):
    p = C.byref(fr.Ssm(A, None, None, channels, states, groups, 1))
    sizes = [fr.lib().frhip_ssm_workspace_bytes(p, n, T) for T in [*range(600), 4096, 100000, 1 << 28] for n in (1, 200)]
    assert sizes == sorted(sizes) and sizes[0::2] == sizes[1::2]
