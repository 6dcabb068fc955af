"""A selective state space layer run as a program runs it: projections, convolution, scan and projection back onto the residual stream, for
two prompts in one call and then token by token, every operator checked against its formula in float64 on the inputs that it had."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from hipref import DevBuf, L, dev, fr, make_weight
from test_gpu_linear import U, act64
from test_gpu_ssm import conv64, half_step, scan64

WIDTH, D, RANK, N, TAPS = 64, 136, 24, 16, 4
BC = RANK + 2 * N  # a row of the second projection: step width, B, C


class Layer:
    def __init__(self, quant, seqs, seed=0):
        g = np.random.default_rng(seed)

        def weight(k, n):
            pw, w = make_weight((g.standard_normal((k, n)) / np.sqrt(k)).astype(np.float16), quant)
            return pw, w.astype(np.float64)
        self.w_in, self.w_bc, self.w_dt, self.w_out = weight(WIDTH, 2 * D), weight(D, BC), weight(RANK, D), weight(D, WIDTH)
        self.taps, self.tap_bias = g.standard_normal((D, TAPS)).astype(np.float32) / 2, g.standard_normal(D).astype(np.float32)
        self.A = (-np.arange(1, N + 1) * g.uniform(0.5, 1.5, (D, N))).astype(np.float32)
        self.skip, self.dt_bias = g.standard_normal(D).astype(np.float32), (g.standard_normal(D) - 3).astype(np.float32)
        self.params = [dev(v) for v in (self.taps, self.tap_bias, self.A, self.skip, self.dt_bias)]
        self.p = fr.Ssm(self.params[2].ptr, self.params[3].ptr, self.params[4].ptr, D, N, 1, 1)
        self.conv_state, self.h = dev(np.zeros((seqs, TAPS - 1, D), np.float16)), dev(np.zeros((seqs, D, N), np.float32))

    def buffers(self, rows, seqs):
        self.xz, self.u, self.bc, self.dt, self.y, self.out = (DevBuf.empty((rows, n), np.float16) for n in (2 * D, D, BC, D, D, WIDTH))
        need = [L().frhip_linear_workspace_bytes(rows, w[0].ref) for w in (self.w_in, self.w_bc, self.w_dt, self.w_out)]
        self.ws = DevBuf(max(need + [L().frhip_ssm_workspace_bytes(C.byref(self.p), seqs, rows), 256]))

    def linear(self, x, ldx, w, y, rows, residual=None, stream=None):
        n = w[0].N
        fr.check(L().frhip_linear(x, ldx, w[0].ref, None, 0, residual, n, y, n, rows, fr.F16, self.ws.ptr, stream), "linear")

    def run(self, x, rows, starts, stream=None):
        """`starts`: prompts; None: a token of each sequence"""
        self.linear(x.ptr, WIDTH, self.w_in, self.xz.ptr, rows, stream=stream)
        conv = (D, TAPS, self.xz.ptr, 2 * D, self.params[0].ptr, self.params[1].ptr, 4, self.conv_state.ptr, self.conv_state.ptr, self.u.ptr, D,
                fr.F16, stream)
        scan = (self.u.ptr, D, self.dt.ptr, D, self.bc.ptr + 2 * RANK, BC, self.bc.ptr + 2 * (RANK + N), BC, self.xz.ptr + 2 * D, 2 * D, self.h.ptr,
                self.h.ptr, self.y.ptr, D, fr.F16)
        if starts is None:
            fr.check(L().frhip_conv_one(rows, *conv), "conv")
        else:
            at = (C.c_int32 * len(starts))(*starts)
            fr.check(L().frhip_conv_seq(len(starts) - 1, at, *conv), "conv")
        self.linear(self.u.ptr, D, self.w_bc, self.bc.ptr, rows, stream=stream)
        self.linear(self.bc.ptr, BC, self.w_dt, self.dt.ptr, rows, stream=stream)
        if starts is None:
            fr.check(L().frhip_ssm_one(C.byref(self.p), rows, *scan, stream), "scan")
        else:
            fr.check(L().frhip_ssm_seq(C.byref(self.p), len(starts) - 1, at, *scan, self.ws.ptr, stream), "scan")
        self.linear(self.y.ptr, D, self.w_out, self.out.ptr, rows, residual=x.ptr, stream=stream)

    def check(self, x, parts, conv0, h0):
        """`parts`: the rows of each sequence; conv0, h0: the states ahead"""
        xz, u, bc, dt, y, out = (b.numpy().astype(np.float64) for b in (self.xz, self.u, self.bc, self.dt, self.y, self.out))

        def close(got, want, tol):
            assert (np.abs(got - want) <= tol + U * np.abs(want) + half_step(np.float16, want)).all()

        def product(got, a, w, res=0.0):
            k = w.shape[0]
            _, tol = act64(a @ w, "none")
            close(got, a @ w + res, tol((k / 32 + 40) * U * (np.abs(a) @ np.abs(w))) + U * np.abs(res))
        product(xz, x.astype(np.float64), self.w_in[1])
        product(bc, u, self.w_bc[1])
        product(dt, bc[:, :RANK], self.w_dt[1])
        product(out, y, self.w_out[1], x.astype(np.float64))
        conv1, h1 = self.conv_state.numpy(), self.h.numpy()
        for i, r in enumerate(parts):
            want, tol, left = conv64(xz[r, :D], self.taps, self.tap_bias, conv0[i], True)
            close(u[r], want, tol)
            assert np.array_equal(conv1[i], left.astype(np.float16))
            want, tol, left, ltol = scan64(u[r], dt[r], bc[r, RANK:RANK + N], bc[r, RANK + N:], xz[r, D:], self.A, self.skip, self.dt_bias, h0[i], 1, True)
            close(y[r], want, tol)
            assert (np.abs(h1[i] - left) <= ltol).all()
        return conv1, h1


@pytest.mark.parametrize("quant", [False, True])
def test_prompts_then_tokens(quant):
    g = np.random.default_rng(1)
    layer = Layer(quant, 2)
    conv, h = layer.conv_state.numpy(), layer.h.numpy()
    x = g.standard_normal((90, WIDTH)).astype(np.float16)
    d = dev(x)
    layer.buffers(90, 2)
    layer.run(d, 90, [0, 83, 90])
    fr.check(L().frhip_device_sync())
    conv, h = layer.check(x, [slice(0, 83), slice(83, 90)], conv, h)
    layer.buffers(2, 2)
    for _ in range(3):
        x = g.standard_normal((2, WIDTH)).astype(np.float16)
        d.nbytes, d.shape, d.dtype = x.nbytes, x.shape, x.dtype
        d.upload(x)
        layer.run(d, 2, None)
        fr.check(L().frhip_device_sync())
        conv, h = layer.check(x, [slice(0, 1), slice(1, 2)], conv, h)


def test_a_captured_token_replays():
    """A layer's token as one graph: every replay takes the states on as an eager call does"""
    g = np.random.default_rng(2)
    eager, graphed = Layer(False, 3), Layer(False, 3)
    st, graph = C.c_void_p(), C.c_void_p()
    fr.check(L().frhip_stream_create(C.byref(st)))
    x = [dev(np.zeros((3, WIDTH), np.float16)) for _ in range(2)]
    eager.buffers(3, 3)
    graphed.buffers(3, 3)
    fr.check(L().frhip_graph_begin(st))
    graphed.run(x[1], 3, None, st)
    fr.check(L().frhip_graph_end(st, C.byref(graph)))
    for _ in range(4):
        v = g.standard_normal((3, WIDTH)).astype(np.float16)
        for b in x:
            b.upload(v)
        fr.check(L().frhip_graph_launch(graph, st))
        eager.run(x[0], 3, None)
        fr.check(L().frhip_stream_sync(st))
        fr.check(L().frhip_device_sync())
        for a, b in ((eager.out, graphed.out), (eager.h, graphed.h), (eager.conv_state, graphed.conv_state)):
            assert np.array_equal(a.numpy(), b.numpy())
    fr.check(L().frhip_graph_destroy(graph))
    fr.check(L().frhip_stream_destroy(st))


def test_two_streams_at_once():
    """Two layers' prompts on streams and workspaces of their own give what each gives alone"""
    g = np.random.default_rng(3)
    x = dev(g.standard_normal((200, WIDTH)).astype(np.float16))
    alone, layers, streams = Layer(True, 1), [Layer(True, 1) for _ in range(2)], [C.c_void_p() for _ in range(2)]
    for a in [alone] + layers:
        a.buffers(200, 1)
    alone.run(x, 200, [0, 200])
    fr.check(L().frhip_device_sync())
    for s in streams:
        fr.check(L().frhip_stream_create(C.byref(s)))
    for _ in range(3):
        for a in layers:
            a.conv_state.upload(np.zeros((1, TAPS - 1, D), np.float16))
            a.h.upload(np.zeros((1, D, N), np.float32))
        for a, s in zip(layers, streams):
            a.run(x, 200, [0, 200], s)
        fr.check(L().frhip_device_sync())
        for a in layers:
            for p, q in ((alone.out, a.out), (alone.h, a.h), (alone.conv_state, a.conv_state)):
                assert np.array_equal(p.numpy(), q.numpy())
    for s in streams:
        fr.check(L().frhip_stream_destroy(s))
