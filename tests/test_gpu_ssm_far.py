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


def test_the_largest_weight_of_codes_with_scales_at_any_address():
    """2^34 codes, ry and my four bytes behind a multiple of 16: expanded a word at a time, in a launch of fewer threads than words.  Rows at the
    begin, the end and on both sides of where the threads begin again are those of a small weight, to the bit; the others hold anything."""
    K, N = 1 << 14, 1 << 20
    rows = np.array([0, 1, 2, (1 << 18) - 1, 1 << 18, (1 << 19) - 1, 1 << 19, 3 << 18, N - 2, N - 1])
    g = np.random.default_rng(6)
    q = g.integers(0, 256, (len(rows), K)).astype(np.uint8)
    mx, rx = (g.uniform(-1, 1, N) / 64).astype(np.float16), (g.uniform(0.5, 1, N) / 64).astype(np.float16)
    my, ry = (g.uniform(-1, 1, K) / 64).astype(np.float16), g.uniform(0.5, 1, K).astype(np.float16)
    off = [dev(np.concatenate([np.zeros(2, np.float16), v])) for v in (my, ry)]
    codes, image = DevBuf(K * N), DevBuf(2 * K * N)
    for r, v in zip(rows, q):
        copy(codes.ptr + int(r) * K, v.ctypes.data, K, H2D)
    dmx, drx = dev(mx), dev(rx)
    w = fr.Weight(codes.ptr, dmx.ptr, drx.ptr, off[0].ptr + 4, off[1].ptr + 4, K, N, fr.U8)
    few = [dev(v) for v in (q, mx[rows], rx[rows], my, ry)]
    small = fr.Weight(*(b.ptr for b in few), K, len(rows), fr.U8)
    want = DevBuf.empty((len(rows), K), np.float16)
    fr.check(L().frhip_dequant_u8(C.byref(small), want.ptr, None))
    want = want.numpy()

    def check():
        fr.check(L().frhip_device_sync())
        for r, v in zip(rows, want):
            got = np.empty(K, np.float16)
            copy(got.ctypes.data, image.ptr + int(r) * K * 2, K * 2, D2H)
            assert np.array_equal(got.view(np.uint16), v.view(np.uint16)), r
    fr.check(L().frhip_dequant_u8(C.byref(w), image.ptr, None))
    check()
    # and as the workspace of a product
    T, form = 1000, (C.c_int * 3)()
    assert L().frhip_linear_form(T, C.byref(w), 256, form) >= 0 and form[2] & 1
    assert L().frhip_linear_workspace_bytes(T, C.byref(w)) == image.nbytes
    clear = np.zeros(K, np.float16)
    for r in rows:
        copy(image.ptr + int(r) * K * 2, clear.ctypes.data, K * 2, H2D)
    x = g.standard_normal((T, K)).astype(np.float16)
    dx, y = dev(x), DevBuf(T * N * 2)
    fr.check(L().frhip_linear(dx.ptr, K, C.byref(w), None, 0, None, 0, y.ptr, N, T, fr.F16, image.ptr, None))
    check()
    for t in (0, T - 1):
        got = np.empty(N, np.float16)
        copy(got.ctypes.data, y.ptr + t * N * 2, N * 2, D2H)
        a, b = x[t].astype(np.float64), want.astype(np.float64)
        tol = (K / 32 + 40) * 2.0 ** -23 * (np.abs(b) @ np.abs(a)) + np.abs(b @ a) * 2.0 ** -11 + 2.0 ** -25
        assert (np.abs(got[rows].astype(np.float64) - b @ a) <= tol).all()
