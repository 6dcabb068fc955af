"""Rows and states of the state space operators that lie more than 4 GiB apart: the same bits as those of the same rows side by side."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from hipref import DevBuf, L, dev, fr, make_weight

PITCH, ROWS = 1 << 22, 600  # of binary16: 5.0e9 bytes
H2D, D2H = fr.H2D, fr.D2H


def copy(to, source, nbytes, kind):
    fr.check(L().frhip_memcpy(to, source, nbytes, kind), "memcpy")


class Far:
    """The rows of `a`, PITCH elements apart"""
    def __init__(self, a):
        a = np.ascontiguousarray(a)
        self.shape, self.dtype, self.row = a.shape, a.dtype, a.shape[1] * a.itemsize
        self.step = PITCH * a.itemsize
        self.buf = DevBuf((len(a) - 1) * self.step + self.row)
        self.ptr = self.buf.ptr
        for i, r in enumerate(a):
            copy(self.ptr + i * self.step, r.ctypes.data, self.row, H2D)

    def numpy(self):
        out = np.empty(self.shape, self.dtype)
        for i, r in enumerate(out):
            copy(r.ctypes.data, self.ptr + i * self.step, self.row, D2H)
        return out


def near_and_far(call, ins, width):
    """call(input, its pitch, y, its pitch) on rows side by side and far apart -> the two y"""
    got = []
    for make, pitch in ((dev, None), (Far, PITCH)):
        x, y = make(ins), make(np.full((len(ins), width), 7, np.float16))
        assert pitch is None or x.buf.nbytes > 1 << 32 and y.buf.nbytes > 1 << 32
        call(x.ptr, pitch or ins.shape[1], y.ptr, pitch or width)
        fr.check(L().frhip_device_sync())
        got.append(y.numpy())
        del x, y
    assert np.isfinite(got[0].astype(np.float32)).all()
    return got


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("act", [0, 4])
def test_product(act, quant):
    g = np.random.default_rng(1)
    K, N = 72, 200
    x = g.standard_normal((ROWS, K)).astype(np.float16)
    w, _ = make_weight((g.standard_normal((K, N)) / 8).astype(np.float16), quant)
    need = L().frhip_linear_workspace_bytes(ROWS, w.ref)
    ws = DevBuf(need) if need else None
    near, far = near_and_far(lambda x, ldx, y, ldy: fr.check(L().frhip_linear(x, ldx, w.ref, None, act, y, ldy, y, ldy, ROWS, fr.F16, ws.ptr if ws else None, None)), x, N)
    assert np.array_equal(near, far)


@pytest.mark.parametrize("one", [False, True])
def test_convolution(one):
    g = np.random.default_rng(2)
    c, W = 75, 4
    x = g.standard_normal((ROWS, c)).astype(np.float16)
    w, n = dev(g.standard_normal((c, W)).astype(np.float32)), ROWS if one else 2
    state = dev(g.standard_normal((n, W - 1, c)).astype(np.float16))
    at = (C.c_int32 * 3)(0, 100, ROWS)
    ends = []

    def call(x, ldx, y, ldy):
        out = DevBuf.empty((n, W - 1, c), np.float16)
        args = (c, W, x, ldx, w.ptr, None, 4, state.ptr, out.ptr, y, ldy, fr.F16, None)
        fr.check(L().frhip_conv_one(n, *args) if one else L().frhip_conv_seq(n, at, *args))
        ends.append(out.numpy())
    near, far = near_and_far(call, x, c)
    assert np.array_equal(near, far) and np.array_equal(*ends)


@pytest.mark.parametrize("one", [False, True])
def test_scan(one):
    g = np.random.default_rng(3)
    d, n = 70, 20
    rows = g.standard_normal((ROWS, 3 * d + 2 * n)).astype(np.float16)  # x, dt, z, B, C
    A, k = dev(-g.uniform(0.5, 4, (d, n)).astype(np.float32)), ROWS if one else 2
    p = fr.Ssm(A.ptr, None, None, d, n, 1, 1)
    state = dev(g.standard_normal((k, d, n)).astype(np.float32))
    at = (C.c_int32 * 3)(0, 100, ROWS)
    ws = DevBuf(L().frhip_ssm_workspace_bytes(C.byref(p), 2, ROWS))
    ends = []

    def call(x, ldx, y, ldy):
        out = DevBuf.empty((k, d, n), np.float32)
        mid = (x, ldx, x + 2 * d, ldx, x + 6 * d, ldx, x + 6 * d + 2 * n, ldx, x + 4 * d, ldx, state.ptr, out.ptr, y, ldy, fr.F16)
        ref = C.byref(p)
        fr.check(L().frhip_ssm_one(ref, k, *mid, None) if one else L().frhip_ssm_seq(ref, k, at, *mid, ws.ptr, None))
        ends.append(out.numpy())
    near, far = near_and_far(call, rows, d)
    assert np.array_equal(near, far) and np.array_equal(*ends)


def test_states_of_many_sequences():
    g = np.random.default_rng(4)
    d, n, rows, last = 1024, 256, 4200, 5  # 4.4e9 bytes of states
    A, state = dev(-g.uniform(0.5, 4, (d, n)).astype(np.float32)), DevBuf(rows * d * n * 4)
    x = g.standard_normal((rows, d)).astype(np.float16)
    bc = g.standard_normal((rows, 2 * n)).astype(np.float16)
    tail = g.standard_normal((last, d, n)).astype(np.float32)
    at = state.ptr + (rows - last) * d * n * 4
    copy(state.ptr, tail.ctypes.data, tail.nbytes, H2D)
    copy(at, tail.ctypes.data, tail.nbytes, H2D)
    p = fr.Ssm(A.ptr, None, None, d, n, 1, 1)

    def run(x, bc, state, count):
        dx, db, dy = dev(x), dev(bc), DevBuf.empty(x.shape, np.float16)
        fr.check(L().frhip_ssm_one(C.byref(p), count, dx.ptr, d, dx.ptr, d, db.ptr, 2 * n, db.ptr + 2 * n, 2 * n, None, 0, state, state, dy.ptr, d, fr.F16, None))
        return dy.numpy()
    y = run(x, bc, state.ptr, rows)
    some = dev(tail)
    want = run(x[-last:], bc[-last:], some.ptr, last)
    left = np.empty_like(tail)
    copy(left.ctypes.data, at, left.nbytes, D2H)
    assert np.isfinite(want.astype(np.float32)).all() and np.array_equal(y[-last:], want) and np.array_equal(left, some.numpy())


def test_more_strips_of_rows_than_sixteen_bits_count():
    T, K, N = 64 * 65536 + 67, 8, 8
    g = np.random.default_rng(5)
    x = g.integers(-8, 9, (T, K)).astype(np.float16)  # sums are exact
    wt = g.integers(-8, 9, (K, N)).astype(np.float16)
    w, _ = make_weight(wt)
    dx, dy = dev(x), DevBuf.empty((T, N), np.float16)
    fr.check(L().frhip_linear(dx.ptr, K, w.ref, None, 0, None, 0, dy.ptr, N, T, fr.F16, None, None))
    assert np.array_equal(dy.numpy(), (x.astype(np.float32) @ wt.astype(np.float32)).astype(np.float16))
