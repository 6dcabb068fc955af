"""The gated delta rule over long prompts: how near every column of a state comes, prompts that go out in several pairs of launches, vectors at the ends of
binary16, rows and states more than 4 GiB apart."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import test_gpu_delta
from hipref import DevBuf, L, dev, fr
from test_gpu_delta import delta_case
from test_gpu_ssm import TYPE, U, half_step, softplus64
from test_gpu_ssm_far import PITCH, Far, copy


def recur64(x, rates, biases, S, heads, kh, dk, dv, eps, scale):
    """One prompt, all its heads at once, token by token in float64 -> y [t][heads][dv], the state behind, and of y the lengths of
    what it is a product of, which it cannot be above"""
    q, k, v, dt, beta = (m.astype(np.float64) for m in x)
    n = len(q)
    q, k = (m.reshape(n, kh, dk) / np.sqrt((m.reshape(n, kh, dk) ** 2).sum(2, keepdims=True) + eps) for m in (q, k))
    q, k = np.repeat(q, heads // kh, 1) * scale, np.repeat(k, heads // kh, 1)
    v, S = v.reshape(n, heads, dv), S.astype(np.float64)
    a, b = np.exp(rates * softplus64(dt + biases)), 1 / (1 + np.exp(-beta))
    y, reach = np.zeros((n, heads, dv)), np.zeros((n, heads, dv))
    for t in range(n):
        S = a[t][:, None, None] * S
        u = b[t][:, None] * (v[t] - np.matmul(k[t][:, None, :], S)[:, 0])
        S = S + k[t][:, :, None] * u[:, None, :]
        y[t] = np.matmul(q[t][:, None, :], S)[:, 0]
        reach[t] = np.sqrt((q[t] ** 2).sum(1))[:, None] * np.sqrt((S * S).sum(1))
    return y, S, reach


def by_columns(heads, kh, dk, dv, lens, dtype, in_place=False):
    """Every column of y and of the state behind, as vectors.  Of a chunk's products each has dk + 64 terms of roundings that know nothing of each other, half a
    dozen of them stand one behind the other, and what a chunk adds is carried on by a recurrence that does not make it longer: so an error's length is near
    sqrt(6 (dk + 64)) U of the column's at a chunk, and sqrt(chunks) of that at the end where nothing is forgotten; twice that is allowed.
    Of y this is relative to the lengths of q and of the state's column, not to y, their product: q (S + E) is off by q E, up to |q| |E| whatever q S is, and
    q S may be next to nothing (in a column of one row it is now and then)."""
    t, code = TYPE[dtype]
    g = np.random.default_rng(dk + heads)
    total = sum(lens)
    silu = lambda m: m / (1 + np.exp(-m))  # noqa: E731
    x = [silu(g.standard_normal((total, n), np.float32)).astype(t) for n in (kh * dk, kh * dk, heads * dv)] + [g.standard_normal((total, heads)).astype(t) for _ in range(2)]
    rates, biases = -np.exp(g.uniform(0, 1, heads)).astype(np.float32), (g.standard_normal(heads) - 5).astype(np.float32)
    S0 = (0.3 * g.standard_normal((len(lens), heads, dk, dv))).astype(np.float32)
    d, ds, dA, db = [dev(v) for v in x], dev(S0), dev(rates), dev(biases)
    do, dy = ds if in_place else DevBuf.empty(S0.shape, np.float32), DevBuf.empty((total, heads * dv), t)
    scale, eps = np.float32(dk ** -0.5), 1e-6
    p = fr.Delta(dA.ptr, db.ptr, heads, kh, dk, dv, scale, eps, 1, 1)
    need = L().frhip_delta_workspace_bytes(C.byref(p), len(lens), total)
    ws = dev(np.full(need + 64, 0x7b, np.uint8))
    at = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    rows = sum(([v.ptr, m.shape[1]] for v, m in zip(d, x)), [])
    fr.check(L().frhip_delta_seq(C.byref(p), len(lens), at.ctypes.data_as(C.c_void_p), *rows, ds.ptr, do.ptr, dy.ptr, heads * dv, code, ws.ptr, None), "delta_seq")
    fr.check(L().frhip_device_sync())
    assert (ws.numpy()[need:] == 0x7b).all()
    y, left = dy.numpy(), do.numpy()
    for i, n in enumerate(lens):
        r = slice(at[i], at[i + 1])
        want, S, reach = recur64([m[r] for m in x], rates.astype(np.float64), biases.astype(np.float64), S0[i], heads, kh, dk, dv, np.float64(np.float32(eps)), np.float64(scale))
        tol = 2 * np.sqrt(6 * (dk + 64) * (n / 64 + 1)) * U

        def length(m, axis):
            return np.sqrt((m * m).sum(axis))
        off, size = length(left[i] - S, 1), length(S, 1)
        assert (off <= tol * size).all(), ("state", i, (off / size).max() / tol)
        got = y[r].reshape(n, heads, dv).astype(np.float64)
        off, size, rounding = length(got - want, 0), length(reach, 0), length(half_step(t, want), 0)
        assert (off <= tol * size + rounding).all(), ("y", i, (off / size).max() / tol)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("size", [(4, 2, 64, 64), (2, 2, 128, 128), (2, 1, 192, 96)])
def test_every_column_of_long_prompts(size, dtype):
    by_columns(*size, [1024, 333, 1], dtype)


@pytest.mark.parametrize("in_place", [False, True])
def test_prompts_in_several_pairs_of_launches(in_place):
    """35 chunks of 13 MB of scratch each, of which a pair of launches takes no more than 20: the first prompt goes on behind one, the second begins there"""
    by_columns(64, 64, 256, 16, [1500, 700], "f32", in_place)


@pytest.mark.parametrize("eps", [0.0, 1e-6])
@pytest.mark.parametrize("n", [3, 100])
@pytest.mark.parametrize("size", [2.0 ** -22, 2.0 ** -14, 2.0 ** 13])
def test_vectors_at_the_ends_of_binary16(size, n, eps, monkeypatch):
    """Subnormal ones, down to a few units, and ones near the largest; where eps is above their squares they do next to nothing"""
    monkeypatch.setattr(test_gpu_delta, "EPS", eps)

    def resize(x, rates, biases, S):
        for m in x[:2]:
            m[:] = np.sign(m) * np.maximum(np.abs(m.astype(np.float64)) * size, 2.0 ** -24)
    delta_case(2, 1, 64, 32, [n], change=resize)


@pytest.mark.parametrize("size", [1e-15, 1e-9, 1e9, 1e15])
@pytest.mark.parametrize("n", [3, 100])
def test_vectors_of_fp32_far_from_one(size, n, monkeypatch):
    monkeypatch.setattr(test_gpu_delta, "EPS", 0.0)

    def resize(x, rates, biases, S):
        for m in x[:2]:
            m *= np.float32(size)
    delta_case(2, 1, 64, 32, [n], "f32", change=resize)


@pytest.mark.parametrize("one", [False, True])
def test_rows_far_apart(one):
    """The same bits as those of the same rows side by side"""
    g = np.random.default_rng(2)
    heads, dk, dv, rows = 2, 32, 32, 600
    x = [g.standard_normal((rows, n)).astype(np.float16) for n in (heads * dk, heads * dk, heads * dv, heads, heads)]
    A, bias = dev(-np.exp(g.uniform(0, 2, heads)).astype(np.float32)), dev((g.standard_normal(heads) - 3).astype(np.float32))
    seqs = rows if one else 2
    state = dev(g.standard_normal((seqs, heads, dk, dv)).astype(np.float32))
    p = fr.Delta(A.ptr, bias.ptr, heads, heads, dk, dv, 0.2, 1e-6, 1, 1)
    at = (C.c_int32 * 3)(0, 90, rows)
    ws, got = DevBuf(L().frhip_delta_workspace_bytes(C.byref(p), 2, rows)), []
    for make, pitch in ((dev, None), (Far, PITCH)):
        d, y, out = [make(m) for m in x], make(np.full((rows, heads * dv), 7, np.float16)), DevBuf.empty((seqs, heads, dk, dv), np.float32)
        args = sum(([b.ptr, pitch or m.shape[1]] for b, m in zip(d, x)), []) + [state.ptr, out.ptr, y.ptr, pitch or heads * dv, fr.F16]
        if one:
            fr.check(L().frhip_delta_one(C.byref(p), rows, *args, None))
        else:
            fr.check(L().frhip_delta_seq(C.byref(p), 2, at, *args, ws.ptr, None))
        fr.check(L().frhip_device_sync())
        got.append((y.numpy(), out.numpy()))
        del d, y, out, args
    assert np.isfinite(got[0][0].astype(np.float32)).all()
    assert all(np.array_equal(a, b) for a, b in zip(*got))


def test_states_of_many_sequences():
    """4.6e9 bytes of states: the last sequences' as alone"""
    g = np.random.default_rng(3)
    heads, dk, dv, rows, last = 16, 256, 256, 1100, 3
    one = heads * dk * dv * 4
    assert rows * one > 1 << 32
    x = [g.standard_normal((rows, n)).astype(np.float16) for n in (heads * dk, heads * dk, heads * dv, heads, heads)]
    p = fr.Delta(None, None, heads, heads, dk, dv, 0.1, 1e-6, 0, 1)
    x[3] = -np.abs(x[3])
    tail = g.standard_normal((last, heads, dk, dv)).astype(np.float32)
    state = DevBuf(rows * one)
    for i in range(0, rows, last):  # (numbers everywhere)
        n = min(last, rows - i)
        copy(state.ptr + i * one, tail.ctypes.data, n * one, fr.H2D)
    at = state.ptr + (rows - last) * one
    copy(at, tail.ctypes.data, tail.nbytes, fr.H2D)

    def run(x, state, count):
        d, y = [dev(m) for m in x], DevBuf.empty((count, heads * dv), np.float16)
        fr.check(L().frhip_delta_one(C.byref(p), count, *sum(([b.ptr, m.shape[1]] for b, m in zip(d, x)), []), state, state, y.ptr, heads * dv, fr.F16, None))
        return y.numpy()
    y = run(x, state.ptr, rows)
    some = dev(tail)
    want = run([m[-last:] for m in x], some.ptr, last)
    left = np.empty_like(tail)
    copy(left.ctypes.data, at, left.nbytes, fr.D2H)
    assert np.isfinite(want.astype(np.float32)).all() and np.array_equal(y[-last:], want) and np.array_equal(left, some.numpy())


@pytest.mark.parametrize("gate", [True, False])
def test_rows_of_the_norms_far_apart(gate):
    g = np.random.default_rng(4)
    rows, cols = 600, 70
    x, z = (g.standard_normal((rows, cols)).astype(np.float16) for _ in range(2))
    p = fr.BlockNorm(None, None, None, None, None, cols, 2, 1, 4, 1.0, 1e-6)
    got = []
    for make, pitch in ((dev, cols), (Far, PITCH)):
        a, b = make(x), make(z)
        y, h = (make(np.full((rows, cols), 7, np.float16)) for _ in range(2))
        if gate:
            fr.check(L().frhip_norm_gate(rows, 7, 10, 1, None, None, 1e-6, a.ptr, pitch, b.ptr, pitch, 4, y.ptr, pitch, fr.F16, None))
        else:
            fr.check(L().frhip_norm_residual(C.byref(p), rows, a.ptr, pitch, b.ptr, pitch, b.ptr, pitch, h.ptr, pitch, fr.F16, y.ptr, pitch, fr.F16, None))
        fr.check(L().frhip_device_sync())
        got.append((y.numpy(), h.numpy()))
        del a, b, y, h
    assert np.isfinite(got[0][0].astype(np.float32)).all() and not (got[0][0] == 7).all()
    assert all(np.array_equal(m, n) for m, n in zip(*got))
