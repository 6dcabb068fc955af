"""The fused norms (norm_gate, norm_residual) against their formulas in float64."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from hipref import DevBuf, L, dev, fr
from test_gpu_ssm import TYPE, U, half_step, silu64

ACT = {"none": 0, "sigmoid": 2, "silu": 4}
NORM = {"none": 0, "rms": 1, "mean": 2}
EPS = 1e-6


def act64(z, err, act):
    """act(z) for z that is off by err, and what it is off by: the exponential by (|z| + 2) units, a reciprocal; slopes of 1 / 4 and 1.1"""
    s = 1 / (1 + np.exp(-z))
    if act == "none":
        return np.ones_like(z) if z is None else z, err
    if act == "sigmoid":
        return s, err / 4 + (np.abs(z) + 6) * U * s
    return silu64(z), 1.1 * err + (np.abs(z) + 6) * U * np.abs(silu64(z))


def norm64(v, err, kind, w, b, eps=EPS):
    """The norm along the last axis of v that is off by err, and what it is off by.  A sum is off by U of its terms' magnitudes for
    every addition that a term goes through, 64 at most (32 in a lane, 6 over a wave, 16 over a workgroup); so is a mean m, and then v - m by that and a unit of
    either; r = 1 / sqrt(q) by half of what q is off by, relative, and two units."""
    if kind == "none":
        return v, err
    n = min(v.shape[-1], 64)
    if kind == "mean":
        m = v.mean(-1, keepdims=True)
        err = err + err.mean(-1, keepdims=True) + (n + 1) * U * np.abs(v).mean(-1, keepdims=True) + U * (np.abs(v) + np.abs(m))
        v = v - m
    q = (v * v).mean(-1, keepdims=True) + eps
    dq = ((2 * np.abs(v) + err) * err).mean(-1, keepdims=True) / q + (n + 4) * U
    y = v / np.sqrt(q)
    err = err / np.sqrt(q) + np.abs(y) * (dq / 2 * (1 + dq) + 3 * U)
    if w is not None:
        y, err = y * w, err * np.abs(w) + U * np.abs(y * w)
    if b is not None:
        y, err = y + b, err + U * (np.abs(y) + np.abs(b))
    return y, err


def close(got, want, tol, t):
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol + half_step(t, want) + 2.0 ** -10 * tol)
    assert not bad.any(), (np.argwhere(bad)[:4], bad.sum(), got[bad][:4], want[bad][:4])


def gate_case(rows, heads, dim, kind="rms", act="silu", dtype="f16", pad=(0, 0, 0), w=True, b=False, z=True, in_place=False, seed=0, x=None, offset=0.0):
    t, code = TYPE[dtype]
    g = np.random.default_rng(seed + rows + dim)
    n = heads * dim
    ldx, ldz, ldy = (n + p for p in pad)
    if in_place:
        ldy = ldx
    x = (g.standard_normal((rows, ldx)) * g.choice([0.01, 1, 30], (rows, 1)) + offset).astype(t) if x is None else x
    zs = g.standard_normal((rows, ldz)).astype(t) * 3
    ws, bs = (1 + g.standard_normal(n)).astype(np.float32), g.standard_normal(n).astype(np.float32)
    dx, dz, dw, db = dev(x), dev(zs), dev(ws), dev(bs)
    dy = dx if in_place else dev(np.full((rows, ldy), 7, t))
    fr.check(L().frhip_norm_gate(rows, heads, dim, NORM[kind], dw.ptr if w else None, db.ptr if b else None, EPS, dx.ptr, ldx, dz.ptr if z else None,
                                 ldz, ACT[act], dy.ptr, ldy, code, None), "norm_gate")
    fr.check(L().frhip_device_sync())
    y = dy.numpy()
    v = x[:, :n].astype(np.float64).reshape(rows, heads, dim)
    want, err = norm64(v, np.zeros_like(v), kind, ws.astype(np.float64).reshape(heads, dim) if w else None, bs.astype(np.float64).reshape(heads, dim) if b else None)
    want, err = want.reshape(rows, n), err.reshape(rows, n)
    if z:
        a, ea = act64(zs[:, :n].astype(np.float64), np.zeros((rows, n)), act)
        want, err = want * a, err * np.abs(a) + np.abs(want) * ea + 2 * U * np.abs(want * a)
    assert np.array_equal(y[:, n:], x[:, n:] if in_place else np.full((rows, ldy - n), 7, t))  # what lies between the rows
    return y[:, :n], want, err, t


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("kind", ["rms", "mean"])
@pytest.mark.parametrize("rows,heads,dim,pad", [
    (1, 1, 1, (0, 0, 0)), (1, 32, 128, (0, 0, 0)), (3, 5, 7, (1, 0, 3)), (65, 3, 64, (0, 8, 0)), (9, 33, 63, (5, 1, 2)), (4, 2, 129, (0, 0, 0)),
    (300, 24, 64, (8, 0, 8)), (2, 3, 256, (0, 0, 0)), (7, 2, 371, (1, 1, 1)), (5, 3, 512, (0, 0, 0)), (6, 1, 1545, (0, 3, 0)), (3, 2, 2049, (0, 0, 0)),
    (3, 1, 4097, (1, 0, 0)), (2, 1, 8193, (0, 0, 0)), (2, 2, 32768, (0, 0, 0)), (40, 1, 2048, (0, 0, 0))])
def test_gate(rows, heads, dim, pad, kind, dtype):
    close(*gate_case(rows, heads, dim, kind, dtype=dtype, pad=pad, b=kind == "mean"))


@pytest.mark.parametrize("act", ["none", "sigmoid", "silu"])
def test_gate_activations_parameters_and_in_place(act):
    close(*gate_case(5, 3, 40, act=act, w=False, b=True, in_place=True))
    close(*gate_case(5, 3, 40, act=act, w=True, dtype="f32", kind="mean", in_place=True, pad=(8, 0, 0)))
    close(*gate_case(33, 4, 64, act=act, w=False, z=False))


def test_gate_of_many_rows():
    close(*gate_case(70000, 1, 8, pad=(0, 0, 0)))


@pytest.mark.parametrize("dim", [64, 300, 5000])
def test_a_mean_far_from_zero_costs_no_digits(dim):
    close(*gate_case(4, 1, dim, kind="mean", dtype="f32", offset=1000.0))


def test_gate_of_zeros_and_of_what_is_not_finite():
    """A head without values is its bias; what is not finite stays in its head"""
    x = np.random.default_rng(0).standard_normal((4, 3 * 40)).astype(np.float32)
    clean, want, err, t = gate_case(4, 3, 40, dtype="f32", x=x.copy(), kind="mean", b=True)
    bad = x.copy()
    bad[1, 40:80], bad[2, 5], bad[3, 100] = 0, np.nan, np.inf
    y, want, err, t = gate_case(4, 3, 40, dtype="f32", x=bad, kind="mean", b=True)
    good = np.ones_like(x, bool)
    good[2, :40] = good[3, 80:] = False
    close(y[good], want[good], err[good], t)
    assert not np.isfinite(y[2, :40]).any() and np.isnan(y[3, 80:]).any()
    same = good.copy()
    same[1, 40:80] = False
    assert np.array_equal(y[same], clean[same])


def residual_case(rows, cols, after="none", before="rms", gate=None, channels=False, scale=1.0, stream="f16", dtype="f16", pad=(0, 0, 0, 0, 0), block=True,
                  one_gate=False, in_place=False, want_h=True, want_y=True, bias=True, seed=0):
    st, scode = TYPE[stream]
    t, code = TYPE[dtype]
    g = np.random.default_rng(seed + rows + cols)
    ldx, ldb, ldg, ldh, ldy = (cols + p for p in pad)
    if in_place:
        ldh = ldx
    x = (g.standard_normal((rows, ldx)) * 2).astype(st)
    bl, gt = g.standard_normal((rows, ldb)).astype(t), g.standard_normal((1 if one_gate else rows, ldg)).astype(t) * 2
    par = [(1 + 0.3 * g.standard_normal(cols)).astype(np.float32) for _ in range(5)]
    dx, dbl, dgt, dpar = dev(x), dev(bl), dev(gt), [dev(v) for v in par]
    dh = dx if in_place else dev(np.full((rows, ldh), 7, st))
    dy = dev(np.full((rows, ldy), 7, t))
    has = [after != "none", after != "none" and bias, before != "none", before != "none" and bias, channels]
    p = fr.BlockNorm(*[d.ptr if h else None for d, h in zip(dpar, has)], cols, NORM[after], NORM[before], ACT[gate or "none"], scale, EPS)
    fr.check(L().frhip_norm_residual(C.byref(p), rows, dx.ptr, ldx, dbl.ptr if block else None, ldb, dgt.ptr if gate else None, 0 if one_gate else ldg,
                                     dh.ptr if want_h else None, ldh, scode, dy.ptr if want_y else None, ldy, code, None), "norm_residual")
    fr.check(L().frhip_device_sync())
    f = [v.astype(np.float64) if h else None for v, h in zip(par, has)]
    h, eh = x[:, :cols].astype(np.float64), np.zeros((rows, cols))
    if block:
        v = bl[:, :cols].astype(np.float64)
        v, ev = norm64(v, np.zeros_like(v), after, f[0], f[1])
        if gate:
            a, ea = act64(gt[:, :cols].astype(np.float64), 0, gate)
            v, ev = v * a, ev * np.abs(a) + np.abs(v) * ea + 2 * U * np.abs(v * a)
        if channels:
            v, ev = v * f[4], ev * np.abs(f[4]) + U * np.abs(v * f[4])
        h, eh = h + scale * v, scale * ev + U * np.abs(h + scale * v)
    y, ey = norm64(h, eh, before, f[2], f[3])
    if want_h:
        got = dh.numpy()
        close(got[:, :cols], h, eh, st)
        assert np.array_equal(got[:, cols:], x[:, cols:] if in_place else np.full((rows, ldh - cols), 7, st))
    if want_y:
        got = dy.numpy()
        close(got[:, :cols], y, ey, t)
        assert (got[:, cols:] == 7).all()
    elif not in_place:
        assert (dy.numpy() == 7).all()


@pytest.mark.parametrize("stream,dtype", [("f16", "f16"), ("f32", "f16"), ("f32", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("rows,cols,kw", [
    (1, 2048, {}), (16, 2048, dict(after="rms", gate="sigmoid", scale=0.5)), (3, 1, dict(after="rms")), (5, 65, dict(after="mean", before="mean", channels=True)),
    (130, 512, dict(gate="silu")), (7, 513, dict(after="rms", gate="none", pad=(1, 2, 3, 4, 5))), (9, 1545, dict(after="mean", before="rms", channels=True)),
    (4, 2049, dict(after="rms", before="mean", gate="sigmoid", channels=True)), (3, 2560, dict(gate="silu", pad=(8, 8, 8, 8, 8))),
    (2, 4097, dict(after="mean", gate="sigmoid")), (2, 8192, dict(after="rms", before="mean", channels=True, gate="silu")),
    (2, 8193, dict(after="rms", gate="sigmoid", channels=True)), (2, 32768, dict(after="mean", before="mean", channels=True, gate="silu"))])
def test_residual(rows, cols, kw, stream, dtype):
    residual_case(rows, cols, stream=stream, dtype=dtype, **kw)


@pytest.mark.parametrize("stream", ["f16", "f32"])
def test_residual_without_some_of_its_parts(stream):
    residual_case(5, 96, stream=stream, block=False)
    residual_case(5, 96, stream=stream, block=False, want_h=False)
    residual_case(5, 96, stream=stream, want_y=False, after="rms")
    residual_case(5, 96, stream=stream, want_h=False, gate="silu", bias=False)
    residual_case(5, 96, stream=stream, before="none")
    residual_case(5, 97, stream=stream, gate="sigmoid", one_gate=True, after="mean")
    residual_case(5, 97, stream=stream, in_place=True, pad=(3, 0, 0, 0, 0), after="rms")


def test_residual_of_many_rows():
    residual_case(9000, 40, after="rms", before="mean", gate="silu", channels=True)


def test_nothing_is_read_or_written_for_no_rows():
    p = fr.BlockNorm(None, None, None, None, None, 64, 0, 1, 0, 1.0, EPS)
    assert L().frhip_norm_residual(C.byref(p), 0, None, 64, None, 64, None, 64, None, 64, 1, None, 64, 1, None) == 0
    assert L().frhip_norm_gate(0, 2, 32, 1, None, None, EPS, None, 64, None, 64, 0, None, 64, 1, None) == 0


def test_captured_calls_replay():
    g = np.random.default_rng(5)
    st, graph = C.c_void_p(), C.c_void_p()
    fr.check(L().frhip_stream_create(C.byref(st)))
    w = dev((1 + g.standard_normal(256)).astype(np.float32))
    x, z, y, h, v, e = (DevBuf.empty((4, 256), np.float16) for _ in range(6))
    p = fr.BlockNorm(w.ptr, None, w.ptr, None, None, 256, 1, 2, 0, 1.0, EPS)

    def run(out_y, out_h, out_v, stream):
        fr.check(L().frhip_norm_gate(4, 4, 64, 1, w.ptr, None, EPS, x.ptr, 256, z.ptr, 256, 4, out_y, 256, fr.F16, stream))
        fr.check(L().frhip_norm_residual(C.byref(p), 4, x.ptr, 256, out_y, 256, None, 0, out_h, 256, fr.F16, out_v, 256, fr.F16, stream))
    fr.check(L().frhip_graph_begin(st))
    run(y.ptr, h.ptr, v.ptr, st)
    fr.check(L().frhip_graph_end(st, C.byref(graph)))
    ey, eh, ev = (DevBuf.empty((4, 256), np.float16) for _ in range(3))
    for _ in range(3):
        x.upload(g.standard_normal((4, 256)).astype(np.float16))
        z.upload(g.standard_normal((4, 256)).astype(np.float16))
        fr.check(L().frhip_graph_launch(graph, st))
        fr.check(L().frhip_stream_sync(st))
        run(ey.ptr, eh.ptr, ev.ptr, None)
        fr.check(L().frhip_device_sync())
        for a, b in ((y, ey), (h, eh), (v, ev)):
            assert np.array_equal(a.numpy(), b.numpy())
    fr.check(L().frhip_graph_destroy(graph))
    fr.check(L().frhip_stream_destroy(st))
