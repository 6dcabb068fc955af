"""frhip_linear (product, bias, activation, residual, one rounding) against the formula in float64."""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from hipref import DevBuf, L, dev, fr, make_weight

U = 2.0 ** -23
ACT = {"none": 0, "sigmoid": 2, "relu2": 3, "silu": 4, "gelu": 5, "softplus": 6}
erfc = np.frompyfunc(math.erfc, 1, 1)


def act64(v, act):
    """The activation, and its tolerance: its slope times the error of v, and the fp32 evaluation's own (an exponential is off by (|v| + 2) U,
    an erfc by the rounding of its argument, v^2 U, and a few units)"""
    if act == "none":
        return v, lambda e: e
    if act == "relu2":
        return np.maximum(v, 0) ** 2, lambda e: 2 * np.abs(v) * e + e * e + U * v * v
    if act == "gelu":
        f = 0.5 * v * erfc(-v / math.sqrt(2)).astype(np.float64)
        return f, lambda e: 1.2 * e + (v * v + 12) * U * np.abs(f) + 2.0 ** -126
    s = 1 / (1 + np.exp(-v))
    f = {"sigmoid": s, "silu": v * s, "softplus": np.logaddexp(0, v)}[act]
    return f, lambda e: 1.1 * e + (np.abs(v) + 12) * U * np.abs(f) + 2.0 ** -126


def case(T, K, N, act="none", bias=False, res=False, out="f16", quant=False, pad=0, in_place=False, seed=0, stream=None, scale=1.0):
    g = np.random.default_rng([T, K, N, seed])
    t, code = (np.float16, fr.F16) if out == "f16" else (np.float32, fr.F32)
    ldx, ldy, ldr = K + 8 * pad, N + pad, N + (pad if in_place else 2 * pad)
    x = g.standard_normal((T, ldx)).astype(np.float16)
    pw, w = make_weight((g.standard_normal((K, N)) * scale / math.sqrt(K)).astype(np.float16), quant)
    b = g.standard_normal(N).astype(np.float32) if bias else None
    y0 = g.standard_normal((T, ldy)).astype(t)
    r = y0 if in_place else g.standard_normal((T, ldr)).astype(t)
    res = res or in_place
    dx, dy = dev(x), dev(y0)
    dr, db = dy if in_place else dev(r), dev(b) if bias else None
    need = L().frhip_linear_workspace_bytes(T, pw.ref)
    ws = DevBuf(need) if need else None
    call = lambda: L().frhip_linear(dx.ptr, ldx, pw.ref, db.ptr if bias else None, ACT[act], dr.ptr if res else None, ldr, dy.ptr, ldy, T,
                                    code, ws.ptr if ws else None, stream)
    fr.check(call(), "linear")
    fr.check(L().frhip_device_sync())
    got = dy.numpy()
    xf, wf = x[:, :K].astype(np.float64), w.astype(np.float64)
    v, mag = xf @ wf, np.abs(xf) @ np.abs(wf)
    if bias:
        v, mag = v + b, mag + np.abs(b)
    # a chain of K / 32 accumulations of sums of 32 exact products (and up to 8 waves' sums), each step within U of the magnitudes
    f, tol = act64(v, act)
    err = tol((K / 32 + 40) * U * mag)
    want = f + (r[:, :N].astype(np.float64) if res else 0)
    err = err + U * np.abs(want) + (np.abs(want) * 2.0 ** -11 + 2.0 ** -25 if out == "f16" else 0)
    bad = ~(np.abs(got[:, :N].astype(np.float64) - want) <= err)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4], got[:, :N][bad][:4], want[bad][:4])
    assert np.array_equal(got[:, N:], y0[:, N:])
    return got, call, dy, y0


# T on both sides of every form's edge, K with and without a rest of 64 and 32, N with ragged ends
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("T,K,N", [(1, 8, 1), (1, 1032, 33), (2, 2048, 130), (3, 40, 7), (4, 64, 64), (5, 256, 515), (16, 104, 48), (17, 2048, 100),
                                   (33, 160, 37), (64, 520, 96), (65, 72, 130), (97, 584, 200), (129, 64, 32), (300, 168, 77), (513, 320, 264),
                                   (520, 256, 1024), (530, 192, 8192), (700, 200, 4000)])
def test_sizes(T, K, N, quant):
    case(T, K, N, quant=quant)
    case(T, K, N, act="silu", bias=True, res=True, out="f32", quant=quant, pad=3, seed=1)


def form(T, K, N, quant):
    out = (C.c_int * 3)()
    return L().frhip_linear_form(T, C.byref(fr.Weight(None, None, None, None, None, K, N, fr.U8 if quant else fr.F16)), 256, out), out[0], out[2]


def test_the_sizes_above_reach_every_form():
    """rows streamed, few rows, tiles of 64, 128 and 256 rows with and without a rest of K, tiles of codes, codes expanded ahead of either"""
    sizes = next(m for m in test_sizes.pytestmark if m.args[0] == "T,K,N").args[1] + [(1030, 1096, 1290), (2050, 520, 4128), (2050, 512, 4128)]
    got = {(f, rows if f != 1 else 0, e, K % 64 != 0) for T, K, N in sizes for q in (False, True) for f, rows, e in [form(T, K, N, q)]}
    for want in [(0, 0, 0, False), (0, 0, 0, True), (1, 0, 0, False), (1, 0, 0, True), (1, 0, 1, True), (2, 64, 0, False), (2, 64, 0, True),
                 (2, 128, 0, False), (2, 128, 0, True), (2, 128, 1, True), (2, 256, 0, False), (2, 256, 0, True), (3, 128, 0, False), (3, 64, 0, False)]:
        assert want in got, (want, sorted(got))


@pytest.mark.parametrize("out", ["f16", "f32"])
@pytest.mark.parametrize("act", sorted(ACT))
@pytest.mark.parametrize("T", [1, 20, 200])
def test_activations(T, act, out):
    case(T, 96, 200, act=act, bias=True, out=out, seed=2, scale=4.0)
    case(T, 96, 200, act=act, res=True, out=out, seed=3)


@pytest.mark.parametrize("out", ["f16", "f32"])
@pytest.mark.parametrize("T", [1, 40, 150])
def test_residual_in_place(T, out):
    case(T, 128, 72, act="gelu", bias=True, out=out, pad=5, in_place=True)


@pytest.mark.parametrize("K", [16, 24, 32, 40, 56, 72, 88, 120, 520, 1032, 1048])
def test_codes_of_rows_of_any_multiple_of_eight(K):
    """The last 16 codes of a row may begin ahead of the last step, and the next row's begin inside them"""
    for T, N in ((1, 33), (20, 130), (70, 17)):
        assert form(T, K, N, True)[0] == 1 and form(T, K, N, True)[2] == 0
        case(T, K, N, quant=True, seed=K)


@pytest.mark.parametrize("T,K,N", [(1030, 1096, 1290), (2050, 520, 4128), (2050, 512, 4128)])
def test_large_products(T, K, N):
    case(T, K, N, act="softplus", bias=True, out="f32", pad=1)
    case(T, K, N, bias=True, res=True)
    case(T, K, N, act="silu", quant=True)


@pytest.mark.parametrize("T,K,N,quant", [(2051, 72, 8192, False), (2050, 64, 8190, False), (2050, 72, 8190, True), (1027, 1000, 8192, False)])
def test_rows_behind_whole_tiles(T, K, N, quant):
    f, rows, how = form(T, K, N, quant)
    assert f == 2 and how == 2 + quant and T % rows
    case(T, K, N, act="silu", bias=True, res=True, quant=quant, pad=3)
    case(T, K, N, out="f32", quant=quant, in_place=True)


def test_what_is_not_finite_stays_in_its_row():
    T, K, N = 70, 200, 90
    g = np.random.default_rng(3)
    for t in (1, 20, T):
        x = g.standard_normal((t, K)).astype(np.float16)
        x[t // 2, 199] = np.nan
        pw, _ = make_weight((g.standard_normal((K, N)) / 14).astype(np.float16))
        dx, dy = dev(x), DevBuf.empty((t, N), np.float16)
        fr.check(L().frhip_linear(dx.ptr, K, pw.ref, None, 3, None, 0, dy.ptr, N, t, fr.F16, None, None))
        y = dy.numpy()
        assert np.isnan(y[t // 2]).all() and np.isfinite(np.delete(y, t // 2, 0)).all()


@pytest.mark.parametrize("T,quant", [(1, False), (20, True), (200, False), (600, True)])
def test_a_captured_product_replays(T, quant):
    st, g = C.c_void_p(), C.c_void_p()
    fr.check(L().frhip_stream_create(C.byref(st)))
    first, call, dy, y0 = case(T, 200, 72, act="silu", bias=True, res=True, quant=quant, stream=st)
    fr.check(L().frhip_graph_begin(st))
    fr.check(call())
    fr.check(L().frhip_graph_end(st, C.byref(g)))
    for _ in range(3):
        dy.upload(y0)
        fr.check(L().frhip_graph_launch(g, st))
        fr.check(L().frhip_stream_sync(st))
        assert np.array_equal(dy.numpy(), first)
    fr.check(L().frhip_graph_destroy(g))
    fr.check(L().frhip_stream_destroy(st))


def test_a_workspace_for_the_most_rows_serves_fewer():
    """2048 x 8192 codes: 1100 rows dequantise on their way, 700 expand; nothing is written behind the workspace that 1100 rows ask for"""
    K, N, guard = 2048, 8192, 1 << 16
    assert form(1100, K, N, True)[2] == 0 and form(700, K, N, True)[2] & 1 == 1
    g = np.random.default_rng(11)
    pw, _ = make_weight((g.standard_normal((K, N)) / math.sqrt(K)).astype(np.float16), True)
    x = g.standard_normal((1100, K)).astype(np.float16)
    need = L().frhip_linear_workspace_bytes(1100, pw.ref)
    assert need >= L().frhip_linear_workspace_bytes(700, pw.ref) >= 2 * K * N
    dx, shared, own = dev(x), dev(np.full(need + guard, 0x5a, np.uint8)), DevBuf(2 * K * N)
    for T in (1100, 700, 3, 1100):
        got = []
        for ws in (shared, own):
            dy = dev(np.full((T, N), 7, np.float16))
            fr.check(L().frhip_linear(dx.ptr, K, pw.ref, None, 0, None, 0, dy.ptr, N, T, fr.F16, ws.ptr, None), "linear")
            got.append(dy.numpy())
        assert np.isfinite(got[0].astype(np.float32)).all() and np.array_equal(*got)
    assert (shared.numpy()[need:] == 0x5a).all()


FAR = np.array([v for m in (0.0, 1e-30, 1e-3, 30, 60, 80, 87, 87.5, 88, 89, 95, 103, 110, 125, 1e3, 1e10, 1e30, 3e38) for v in (m, -m)], np.float32)


@pytest.mark.parametrize("out", ["f16", "f32"])
@pytest.mark.parametrize("act", sorted(ACT))
@pytest.mark.parametrize("T", [1, 20, 200])
def test_activations_far_from_zero(T, act, out):
    """v = bias exactly.  A sigmoid below the normal numbers may be 0 (its reciprocal is subnormal), which silu multiplies by |v| <= 104."""
    N, t = len(FAR), np.float16 if out == "f16" else np.float32
    pw, _ = make_weight(np.zeros((8, N), np.float16))
    dx, db, dy = dev(np.zeros((T, 8), np.float16)), dev(FAR), DevBuf.empty((T, N), t)
    fr.check(L().frhip_linear(dx.ptr, 8, pw.ref, db.ptr, ACT[act], None, 0, dy.ptr, N, T, fr.F16 if out == "f16" else fr.F32, None, None))
    with np.errstate(over="ignore"):
        v = FAR.astype(np.float64)
        f, tol = act64(v, act)
        tol = tol(0.0) + np.where((v < -87) & (v > -104), -v, 1) * 2.0 ** -126 + (np.abs(f) * 2.0 ** -11 + 2.0 ** -25 if out == "f16" else np.abs(f) * 2.0 ** -24)
        rounded = f.astype(t)
    got = dy.numpy()
    for row in got:
        bad = ~(np.abs(row.astype(np.float64) - f) <= tol) & (row != rounded)  # what overflows is infinite in both
        assert not bad.any(), (v[bad], row[bad], f[bad])


@pytest.mark.parametrize("T,K,N,quant", [(1, 200, 90, False), (2, 1032, 33, False), (1, 200, 90, True), (20, 200, 90, False), (48, 72, 130, True), (300, 168, 80, False),
                                         (200, 2048, 8192, True), (1030, 200, 4000, False), (700, 200, 4000, True)])
@pytest.mark.parametrize("act", sorted(ACT))
def test_infinities_are_those_of_the_formula(act, T, K, N, quant):
    """An infinite x gives infinite sums of its weights' signs; what multiplies minus infinity by the zero that its sigmoid or erfc is may be 0 or a NaN"""
    g = np.random.default_rng(12)
    w = g.uniform(0.25, 1, (K, N)) * np.where(g.random(N) < 0.5, -1, 1)  # the codes' signs are the weights'
    pw, wf = make_weight(w.astype(np.float16), quant)
    assert (np.sign(wf) == np.sign(w)).all()
    x = (g.standard_normal((T, K)) / K).astype(np.float16)
    where = [(0, K - 1, np.inf), (T // 2, 0, -np.inf), (T - 1, K - 9, np.inf)]
    for r, k, v in where:
        x[r] = 0
        x[r, k] = v
    dx, out = dev(x), []
    need = L().frhip_linear_workspace_bytes(T, pw.ref)
    ws = DevBuf(need) if need else None
    for code, t in ((fr.F16, np.float16), (fr.F32, np.float32)):
        dy = DevBuf.empty((T, N), t)
        fr.check(L().frhip_linear(dx.ptr, K, pw.ref, None, ACT[act], None, 0, dy.ptr, N, T, code, ws.ptr if ws else None, None))
        y = dy.numpy()
        last = {r: v for r, _, v in where}
        for r, v in last.items():
            up = np.sign(w[0]) * np.sign(v) > 0
            assert (y[r, up] == (1 if act == "sigmoid" else np.inf)).all(), (code, r)
            down = y[r, ~up].astype(np.float64)
            if act == "none":
                assert (down == -np.inf).all()
            else:
                assert ((np.abs(down) <= 2.0 ** -126) | (np.isnan(down) if act in ("silu", "gelu") else False)).all(), (code, r, down)
        assert np.isfinite(np.delete(y, list(last), 0).astype(np.float32)).all()


@pytest.mark.parametrize("T", [1, 20, 200])
def test_rows_of_fp32_beside_those_of_x(T):
    """One buffer of 256 bytes a row: 64 binary16, then 32 fp32 that receive their product"""
    g = np.random.default_rng(T)
    buf = g.standard_normal((T, 128)).astype(np.float16)
    pw, _ = make_weight((g.standard_normal((64, 32)) / 8).astype(np.float16))
    near, d, dy = dev(np.ascontiguousarray(buf[:, :64])), dev(buf), DevBuf.empty((T, 32), np.float32)
    fr.check(L().frhip_linear(near.ptr, 64, pw.ref, None, 0, None, 0, dy.ptr, 32, T, fr.F32, None, None))
    fr.check(L().frhip_linear(d.ptr, 128, pw.ref, None, 0, None, 0, d.ptr + 128, 64, T, fr.F32, None, None))
    got = d.numpy()
    assert np.array_equal(got[:, :64], buf[:, :64]) and np.array_equal(np.ascontiguousarray(got[:, 64:]).view(np.float32), dy.numpy())
