"""The selective state space operators (short convolution, selective scan) against their formulas in float64."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from hipref import DevBuf, L, dev, fr

U = 2.0 ** -23  # the unit of one fp32 operation of the device: its exp2 and reciprocal are within it, correctly rounded ones within half
TYPE = {"f16": (np.float16, fr.F16), "f32": (np.float32, fr.F32)}
GUARD = 3  # rows ahead of the first prompt and behind the last


def half_step(dtype, y):
    """What one rounding to the type is off by at most"""
    return np.abs(y) * 2.0 ** -11 + 2.0 ** -25 if dtype == np.float16 else np.abs(y) * 2.0 ** -24 + 2.0 ** -149


def seq_table(lens):
    at = np.concatenate([[GUARD], GUARD + np.cumsum(lens)]).astype(np.int32)
    return at, at.ctypes.data_as(C.c_void_p)


def silu64(v):
    return v / (1 + np.exp(-v))


def silu_error(v, err):
    """Of silu(v) in fp32 where v is off by `err`: its slope is 1.1 at most, its exponential off by (|v| + 2) units, relative"""
    return 1.1 * err + (np.abs(v) + 6) * U * np.abs(silu64(v))


# ---- convolution ---------------------------------------------------------------------------------------------------
def conv64(x, w, bias, state, act):
    """x [t][c], state [W-1][c] -> y, its tolerance before rounding, the state behind"""
    W = w.shape[1]
    past = np.concatenate([state, x]).astype(np.float64)
    win = np.stack([past[j:j + len(x)] for j in range(W)], 2) * w.astype(np.float64)
    b = bias.astype(np.float64) if bias is not None else np.zeros(w.shape[0])
    v = win.sum(2) + b
    err = (np.abs(win).sum(2) + np.abs(b)) * W * U  # W fused multiply-adds, each within half a unit of a partial sum
    return (silu64(v), silu_error(v, err), past[len(x):]) if act else (v, err, past[len(x):])


def conv_case(seed, c, W, lens, dtype, ldx, bias=True, act=True, one=False, in_place=False, stream=None):
    t, code = TYPE[dtype]
    g = np.random.default_rng(seed)
    n, total = len(lens), int(sum(lens)) + (0 if one else 2 * GUARD)
    x = g.standard_normal((total, ldx)).astype(t)
    w = g.standard_normal((c, W)).astype(np.float32)
    b = g.standard_normal(c).astype(np.float32) if bias else None
    state = g.standard_normal((n, W - 1, c)).astype(t)
    ldy = c + 5
    mark = np.full((total, ldy), 7, t)
    dx, dw, ds, dy = dev(x), dev(w), dev(state), dev(mark)
    db = dev(b) if bias else None
    do = ds if in_place else dev(np.full_like(state, 9))
    args = (c, W, dx.ptr, ldx, dw.ptr, db.ptr if bias else None, 4 if act else 0, ds.ptr, do.ptr, dy.ptr, ldy, code, stream)
    at, ptr = seq_table(lens)
    if one:
        fr.check(L().frhip_conv_one(n, *args), "conv_one")
        at = np.arange(n + 1)
    else:
        fr.check(L().frhip_conv_seq(n, ptr, *args), "conv_seq")
    fr.check(L().frhip_device_sync())
    y, left = dy.numpy(), do.numpy()
    want = mark.astype(np.float64)
    tol = np.zeros_like(want)
    for i in range(n):
        a, e = at[i], at[i + 1]
        want[a:e, :c], tol[a:e, :c], end = conv64(x[a:e, :c], w, b, state[i], act)
        assert np.array_equal(left[i], end.astype(t)), (i, lens[i])
    bad = np.abs(y.astype(np.float64) - want) > tol + np.where(tol > 0, half_step(t, want) + U * np.abs(want), 0)
    assert not bad.any(), (np.argwhere(bad)[:4], bad.sum())
    return y


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("c,W,lens", [(1, 2, [1]), (7, 4, [5]), (64, 3, [0]), (65, 4, [1, 2, 3, 4, 0, 16, 17]), (96, 2, [15, 16, 33]),
                                      (2049, 4, [40, 1]), (520, 3, [129])])
def test_conv_seq(c, W, lens, dtype):
    conv_case(c, c, W, lens, dtype, ldx=c + c % 3)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("c,W,rows", [(1, 2, 1), (13, 3, 5), (768, 4, 1), (770, 4, 33), (64, 2, 300)])
def test_conv_one(c, W, rows, dtype):
    conv_case(c + rows, c, W, [1] * rows, dtype, ldx=2 * c, one=True)


@pytest.mark.parametrize("one", [False, True])
def test_conv_without_bias_or_activation_and_with_its_state_in_place(one):
    conv_case(1, 40, 4, [1, 1, 1] if one else [1, 2, 0, 50], "f16", 41, bias=False, act=False, one=one, in_place=True)
    conv_case(2, 40, 3, [1, 1, 1] if one else [1, 2, 0, 50], "f32", 40, one=one, in_place=True)


def test_conv_of_more_prompts_than_a_launch_holds():
    conv_case(3, 24, 4, [i % 5 for i in range(300)], "f16", 24)


# ---- scan ----------------------------------------------------------------------------------------------------------
def softplus64(v):
    return np.logaddexp(0, v)


def scan64(x, dt, B, Cv, z, A, D, bias, state, groups, softplus):
    """Everything in float64; returns y, its tolerance before rounding, the state behind and its tolerance.

    The tolerances follow the fp32 evaluation.  With U per operation: the step width is off by dd = (|v| + 10) U relative (softplus: an
    exponential whose argument is rounded, a reciprocal, a polynomial); a decay exp(a) by (dd + 3 U)|a| + 3 U; a state by the
    decayed error of the one before, its decay's, its input's and its own rounding, of the sum M of the terms' magnitudes; the
    sums of step widths that join chunks by T U, which moves exp(-s) by T U / e at most; an output by N + 2 units of its terms."""
    T, d = x.shape
    n = A.shape[1]
    f = np.float64
    v = dt.astype(f) + (bias.astype(f) if bias is not None else 0)
    step = softplus64(v) if softplus else v
    dd = (np.abs(v) + 10) * U if softplus else np.full_like(v, U)
    Bc, Cc = (np.repeat(m.astype(f).reshape(T, groups, n), d // groups, 1) for m in (B, Cv))
    A = A.astype(f)
    h, E, M = state.astype(f), np.zeros((d, n)), np.abs(state.astype(f))
    y, tol = np.zeros((T, d)), np.zeros((T, d))
    for t in range(T):
        a = step[t][:, None] * A
        decay, b = np.exp(a), (step[t] * x[t].astype(f))[:, None] * Bc[t]
        da = (dd[t][:, None] + 3 * U) * np.abs(a) + 3 * U
        E = decay * (E + da * M) + (dd[t][:, None] + 3 * U) * np.abs(b)
        h, M = decay * h + b, decay * M + np.abs(b)
        E = E + U * M
        skip = (D.astype(f) if D is not None else np.zeros(d)) * x[t]
        terms = (np.abs(Cc[t]) * M).sum(1) + np.abs(skip)
        y[t] = (Cc[t] * h).sum(1) + skip
        tol[t] = (np.abs(Cc[t]) * (E + 0.37 * T * U * M)).sum(1) + (n + 2) * U * terms
    if z is not None:
        zf = z.astype(f)
        tol = np.abs(silu64(zf)) * tol + np.abs(y) * silu_error(zf, 0)
        y = y * silu64(zf)
    return y, tol, h, E + 0.37 * T * U * M


class Scan:
    def __init__(self, seed, d, n, lens, dtype="f16", groups=1, gate=True, skip=True, bias=True, softplus=True, one=False, in_place=False,
                 spread=1.0):
        t, self.code = TYPE[dtype]
        g = np.random.default_rng(seed)
        self.t, self.d, self.n, self.groups, self.lens, self.one = t, d, n, groups, lens, one
        total = int(sum(lens)) + (0 if one else 2 * GUARD)
        self.ld = {"x": d + 3, "dt": d, "bc": 2 * groups * n + 1, "z": d + 8, "y": d + 1}
        self.x = g.standard_normal((total, self.ld["x"])).astype(t)
        self.dt = (g.standard_normal((total, d)) * spread if softplus else g.uniform(0, 0.5, (total, d))).astype(t)
        self.bc = g.standard_normal((total, self.ld["bc"])).astype(t)
        self.z = g.standard_normal((total, self.ld["z"])).astype(t) if gate else None
        self.A = (-np.arange(1, n + 1) * g.uniform(0.5, 1.5, (d, n))).astype(np.float32)
        self.D = g.standard_normal(d).astype(np.float32) if skip else None
        self.bias = (g.standard_normal(d) - 2).astype(np.float32) if bias and softplus else None
        self.state = g.standard_normal((len(lens), d, n)).astype(np.float32)
        self.mark = np.full((total, self.ld["y"]), 7, t)
        self.softplus = softplus
        self.in_place = in_place
        self.buf = {k: dev(v) for k, v in (("x", self.x), ("dt", self.dt), ("bc", self.bc), ("z", self.z), ("A", self.A), ("D", self.D),
                                           ("bias", self.bias), ("state", self.state), ("y", self.mark)) if v is not None}
        self.out = self.buf["state"] if in_place else dev(np.full_like(self.state, 9))
        ptr = lambda k: self.buf[k].ptr if k in self.buf else None
        self.p = fr.Ssm(ptr("A"), ptr("D"), ptr("bias"), d, n, groups, int(softplus))
        need = 0 if one else L().frhip_ssm_workspace_bytes(C.byref(self.p), len(lens), int(sum(lens)))
        self.ws = DevBuf(need) if need else None

    def call(self, stream=None):
        b, e = self.buf, np.dtype(self.t).itemsize
        self.at, table = seq_table(self.lens)
        mid = (b["x"].ptr, self.ld["x"], b["dt"].ptr, self.ld["dt"], b["bc"].ptr, self.ld["bc"], b["bc"].ptr + self.groups * self.n * e,
               self.ld["bc"], b["z"].ptr if "z" in b else None, self.ld["z"], b["state"].ptr, self.out.ptr, b["y"].ptr, self.ld["y"], self.code)
        ref = C.byref(self.p)
        if self.one:
            self.at = np.arange(len(self.lens) + 1)
            return L().frhip_ssm_one(ref, len(self.lens), *mid, stream)
        return L().frhip_ssm_seq(ref, len(self.lens), table, *mid, self.ws.ptr if self.ws else None, stream)

    def check(self):
        fr.check(L().frhip_device_sync())
        y, left = self.buf["y"].numpy(), self.out.numpy()
        want, tol = self.mark.astype(np.float64), np.zeros(self.mark.shape)
        gn = self.groups * self.n
        for i in range(len(self.lens)):
            a, e = self.at[i], self.at[i + 1]
            want[a:e, :self.d], tol[a:e, :self.d], h, ht = scan64(
                self.x[a:e, :self.d], self.dt[a:e], self.bc[a:e, :gn], self.bc[a:e, gn:2 * gn],
                self.z[a:e, :self.d] if self.z is not None else None, self.A, self.D, self.bias, self.state[i], self.groups, self.softplus)
            bad = np.abs(left[i] - h) > ht
            assert not bad.any(), ("state", i, self.lens[i], bad.sum(), np.argwhere(bad)[:4])
        wide = tol + np.where(tol > 0, half_step(self.t, want) + U * np.abs(want), 0)
        bad = np.abs(y.astype(np.float64) - want) > wide
        assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4])
        return y, left


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("d,n,groups,lens", [(1, 1, 1, [1]), (65, 3, 1, [9]), (64, 16, 1, [0]), (130, 5, 2, [8, 0, 17, 1]),
                                             (96, 16, 1, [700]), (48, 24, 3, [33, 40]), (70, 64, 1, [260, 3]), (10, 130, 2, [50]), (33, 256, 1, [70]),
                                             (20, 100, 2, [40, 3]), (65, 40, 1, [21]),
                                             (300, 8, 1, [16, 15, 250]),
                                             (70, 16, 1, [32, 17, 0, 31]), (130, 64, 1, [32]), (66, 16, 1, [33])])
def test_scan_seq(d, n, groups, lens, dtype):
    s = Scan(d * n, d, n, lens, dtype, groups)
    fr.check(s.call(), "ssm_seq")
    s.check()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("d,n,groups,rows", [(1, 1, 1, 1), (65, 3, 1, 2), (768, 16, 1, 1), (96, 16, 3, 7), (40, 24, 2, 5), (33, 64, 1, 3), (10, 130, 2, 4),
                                             (17, 256, 1, 9), (520, 8, 1, 40)])
def test_scan_one(d, n, groups, rows, dtype):
    s = Scan(d * n + rows, d, n, [1] * rows, dtype, groups, one=True)
    fr.check(s.call(), "ssm_one")
    s.check()


@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("kw", [dict(gate=False), dict(skip=False), dict(bias=False), dict(softplus=False), dict(in_place=True),
                                dict(gate=False, skip=False, bias=False, in_place=True), dict(spread=12.0)])
def test_scan_options(kw, one):
    s = Scan(5, 72, 16, [1] * 4 if one else [200, 0, 31], "f16", **kw, one=one)
    fr.check(s.call())
    s.check()
    s = Scan(6, 72, 16, [1] * 4 if one else [200, 0, 31], "f32", **kw, one=one)
    fr.check(s.call())
    s.check()


def test_scan_of_more_prompts_than_a_launch_holds():
    s = Scan(7, 20, 4, [i % 40 for i in range(150)], "f16")
    fr.check(s.call())
    s.check()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_a_prompt_in_pieces_and_token_by_token(dtype):
    """The state that one call leaves is the one that the next takes: 90 rows at once, as 50 + 40, and the last 40 one by one."""
    whole = Scan(8, 200, 16, [90], dtype)
    fr.check(whole.call())
    y, left = whole.check()
    b, e = whole.buf, np.dtype(whole.t).itemsize
    out = dev(whole.mark)
    st = dev(whole.state)

    def run(call, row, head, *tail):
        at = lambda k: b[k].ptr + row * whole.ld[k] * e
        fr.check(call(C.byref(whole.p), *head, at("x"), whole.ld["x"], at("dt"), whole.ld["dt"], at("bc"), whole.ld["bc"], at("bc") + 16 * e,
                      whole.ld["bc"], at("z"), whole.ld["z"], st.ptr, st.ptr, out.ptr + row * whole.ld["y"] * e, whole.ld["y"], whole.code, *tail))
    run(L().frhip_ssm_seq, GUARD, (1, (C.c_int32 * 2)(0, 50)), whole.ws.ptr, None)
    for r in range(40):
        run(L().frhip_ssm_one, GUARD + 50 + r, (1,), None)
    fr.check(L().frhip_device_sync())
    got = Scan(8, 200, 16, [90], dtype)  # the same numbers: its check compares with float64
    got.at = whole.at
    got.buf["y"], got.out = out, st
    got.check()


def test_a_captured_scan_and_convolution_replay():
    s = Scan(9, 130, 16, [120, 7], "f16")
    st = C.c_void_p()
    fr.check(L().frhip_stream_create(C.byref(st)))
    g = C.c_void_p()
    fr.check(s.call(st))
    fr.check(L().frhip_stream_sync(st))
    first = s.check()
    fr.check(L().frhip_graph_begin(st))
    fr.check(s.call(st))
    fr.check(L().frhip_graph_end(st, C.byref(g)))
    for _ in range(3):
        s.buf["y"].upload(s.mark)
        s.out.upload(np.full_like(s.state, 9))
        fr.check(L().frhip_graph_launch(g, st))
        fr.check(L().frhip_stream_sync(st))
        again = s.check()
        assert all(np.array_equal(a, b) for a, b in zip(first, again))
        conv_case(4, 40, 4, [1, 2, 0, 50], "f16", 41, stream=st)
    fr.check(L().frhip_graph_destroy(g))
    fr.check(L().frhip_stream_destroy(st))


def test_what_is_not_finite_stays_in_its_channel():
    s = Scan(10, 96, 16, [60], "f16")
    s.x[GUARD + 20, 5], s.x[GUARD + 30, 70], s.dt[GUARD + 40, 9] = np.inf, np.nan, -np.inf
    s.buf["x"].upload(s.x)
    s.buf["dt"].upload(s.dt)
    fr.check(s.call())
    fr.check(L().frhip_device_sync())
    y, left = s.buf["y"].numpy()[GUARD:GUARD + 60, :96], s.out.numpy()[0]
    ok = np.ones((60, 96), bool)
    ok[20:, 5] = ok[30:, 70] = False
    assert np.isfinite(y[ok].astype(np.float32)).all() and not np.isfinite(y[~ok].astype(np.float32)).any()
    fine = np.isfinite(left).all(1)
    assert fine.sum() == 94 and not fine[5] and not fine[70]  # a step of width zero (softplus(-inf)) is fine


@pytest.mark.parametrize("one", [False, True])
def test_a_rate_of_minus_infinity_forgets(one):
    s = Scan(13, 70, 16, [1] * 5 if one else [90, 0, 7], "f32", one=one)
    s.A[:, 3] = -np.inf
    s.buf["A"].upload(s.A)
    s.A[:, 3] = -1e30  # for every step width here the decay is zero as well
    fr.check(s.call())
    s.check()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("softplus", [False, True])
@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("n", [16, 6])
def test_a_step_of_width_zero_keeps_the_state_at_any_rate(n, one, softplus, dtype):
    """Padding tokens: rates of minus infinity, and finite ones whose product with log2(e) is none, times zero"""
    s = Scan(14, 70, n, [1] * 5 if one else [90, 0, 7], dtype, one=one, softplus=softplus)
    s.A[:, 2], s.A[:, 5] = -np.inf, -3e38
    s.buf["A"].upload(s.A)
    s.A[:, 2] = -1e30  # for every step width here the decay is 0 or 1 as well
    none = [0, 3] if one else [GUARD, GUARD + 3, GUARD + 15, GUARD + 16, *range(GUARD + 30, GUARD + 50), GUARD + 89, GUARD + 90, GUARD + 96]
    s.dt[none] = -60000 if softplus else 0
    s.dt[:, 7] = -60000 if softplus else 0  # a channel of nothing else
    s.buf["dt"].upload(s.dt)
    fr.check(s.call())
    y, left = s.check()
    assert np.isfinite(y.astype(np.float32)).all() and all(np.array_equal(a[7], b[7]) for a, b in zip(left, s.state))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("what", ["x", "dt"])
@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("n", [1, 3, 6, 16, 24, 40, 100, 130, 256])
def test_an_infinite_input_is_infinity_whatever_the_states(n, one, what, dtype):
    """Everything positive: h is infinite from that token on and so is y; a form's states beyond `states` have no part in it"""
    s = Scan(15, 70, n, [1] * 5 if one else [60, 0, 7], dtype, one=one)
    for v in (s.x, s.bc, s.z, s.D, s.state):
        np.abs(v, out=v)
    s.A = (s.A / (16 * n)).astype(np.float32)  # decays of 60 rows are far from zero
    for k in ("x", "bc", "z", "D", "state", "A"):
        s.buf[k].upload(getattr(s, k))
    start = s.state.copy()
    fr.check(s.call())
    clean = [v.copy() for v in s.check()]
    rows = [1, 2] if one else [GUARD + 19, GUARD + 62]  # in the second chunk of the first prompt; in the last prompt
    v = getattr(s, what)
    for r, c in zip(rows, (5, 69)):
        v[r, c] = np.inf
    s.buf[what].upload(v)
    s.buf["state"].upload(start)
    s.buf["y"].upload(s.mark)
    fr.check(s.call())
    fr.check(L().frhip_device_sync())
    y, left = s.buf["y"].numpy(), s.out.numpy()
    for r, c in zip(rows, (5, 69)):
        i = int(np.searchsorted(s.at, r, side="right")) - 1
        clean[0][r:s.at[i + 1], c] = np.inf
        clean[1][i, c] = np.inf
    assert np.array_equal(y, clean[0]) and np.array_equal(left, clean[1])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("d,n,groups,lens", [(130, 129, 1, [1000]), (70, 256, 1, [700, 130]), (200, 200, 2, [300, 0, 40, 600]), (640, 256, 1, [200]), (65, 128, 1, [400, 33])])
def test_many_states_over_many_chunks(d, n, groups, lens, dtype):
    s = Scan(d + n, d, n, lens, dtype, groups)
    cut, at = (C.c_int * 3)(), np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    assert L().frhip_ssm_cut(C.byref(s.p), len(lens), at.ctypes.data_as(C.c_void_p), 256, cut) == 0 and cut[1] > len(lens) + 4
    fr.check(s.call(), "ssm_seq")
    y, left = s.check()
    assert np.isfinite(y.astype(np.float32)).all() and np.isfinite(left).all()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("one", [False, True])
def test_gates_far_from_zero(one, dtype):
    """silu(z) of a convolution's sums and of a scan's gates where its exponential leaves fp32: what is below the normal numbers may be 0"""
    t = TYPE[dtype][0]
    far = np.array([v for m in (30, 60, 80, 87, 87.5, 88, 89, 95, 103, 110, 125, 1e3, 6e4, 1e30, 3e38) for v in (m, -m) if dtype == "f32" or m < 65504], t)
    c = len(far)
    with np.errstate(over="ignore"):
        want, tol = silu64(far.astype(np.float64)), silu_error(far.astype(np.float64), 0)
    tol = np.where(np.isfinite(tol), tol, 0) + half_step(t, want) + np.where((far < -87) & (far > -104), -far.astype(np.float64), 1) * 2.0 ** -126

    def close(rows):
        bad = ~(np.abs(rows.astype(np.float64) - want) <= tol)
        assert not bad.any(), (np.argwhere(bad)[:4], rows[bad][:4])
    # a convolution that takes x as it is
    x = np.tile(far, (9, 1))
    w = np.zeros((c, 4), np.float32)
    w[:, 3] = 1
    dx, dw, st, dy = dev(x), dev(w), dev(np.zeros((9, 3, c), t)), DevBuf.empty((9, c), t)
    args = (c, 4, dx.ptr, c, dw.ptr, None, 4, st.ptr, st.ptr, dy.ptr, c, TYPE[dtype][1], None)
    fr.check(L().frhip_conv_one(9, *args) if one else L().frhip_conv_seq(1, (C.c_int32 * 2)(0, 9), *args))
    close(dy.numpy())
    # a scan whose y is 1 ahead of the gate: D x, an empty state and no input
    zero, ones = dev(np.zeros((9, c), t)), dev(np.ones((9, c), t))
    A, D, h, dy = dev(-np.ones((c, 4), np.float32)), dev(np.ones(c, np.float32)), dev(np.zeros((9, c, 4), np.float32)), DevBuf.empty((9, c), t)
    p = fr.Ssm(A.ptr, D.ptr, None, c, 4, 1, 0)
    mid = (ones.ptr, c, zero.ptr, c, zero.ptr, c, zero.ptr, c, dx.ptr, c, h.ptr, h.ptr, dy.ptr, c, TYPE[dtype][1])
    ws = DevBuf(max(L().frhip_ssm_workspace_bytes(C.byref(p), 1, 9), 16))
    fr.check(L().frhip_ssm_one(C.byref(p), 9, *mid, None) if one else L().frhip_ssm_seq(C.byref(p), 1, (C.c_int32 * 2)(0, 9), *mid, ws.ptr, None))
    close(dy.numpy())


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_outputs_of_finite_inputs_are_numbers(dtype):
    """Every size of the tests above: the comparisons that they make let a NaN pass"""
    sizes = lambda test, names: next(m for m in test.pytestmark if m.args[0] == names).args[1]
    for d, n, groups, lens in sizes(test_scan_seq, "d,n,groups,lens"):
        s = Scan(d * n, d, n, lens, dtype, groups)
        fr.check(s.call())
        assert all(np.isfinite(v.numpy().astype(np.float32)).all() for v in (s.buf["y"], s.out)), (d, n, lens)
    for d, n, groups, rows in sizes(test_scan_one, "d,n,groups,rows"):
        s = Scan(d * n + rows, d, n, [1] * rows, dtype, groups, one=True)
        fr.check(s.call())
        assert all(np.isfinite(v.numpy().astype(np.float32)).all() for v in (s.buf["y"], s.out)), (d, n, rows)
    for c, W, lens in sizes(test_conv_seq, "c,W,lens"):
        assert np.isfinite(conv_case(c, c, W, lens, dtype, ldx=c + c % 3).astype(np.float32)).all(), (c, W, lens)
    for c, W, rows in sizes(test_conv_one, "c,W,rows"):
        assert np.isfinite(conv_case(c + rows, c, W, [1] * rows, dtype, ldx=2 * c, one=True).astype(np.float32)).all(), (c, W, rows)
