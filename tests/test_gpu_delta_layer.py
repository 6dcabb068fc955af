"""A gated delta-rule layer run as a program runs it: norm, projection, convolution, delta rule, gated norm, projection back and the residual with
both norms, for two prompts in one call and then token by token, every operator checked against its formula in float64 on the inputs that it had."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from hipref import DevBuf, L, dev, fr, make_weight
from test_gpu_delta import either
from test_gpu_linear import act64 as linear64
from test_gpu_norm import EPS, act64, norm64
from test_gpu_ssm import U, conv64, half_step

WIDTH, HEADS, KEY_HEADS, DK, DV, TAPS = 64, 8, 2, 32, 24, 4
KN, VN = KEY_HEADS * DK, HEADS * DV
MIX = 2 * KN + VN              # what the convolution goes over: q, k, v
ROW = MIX + VN + 2 * HEADS     # of the first projection: those, the gate, dt, beta
H1 = np.float16


class Layer:
    def __init__(self, quant, seqs, seed=0):
        g = np.random.default_rng(seed)

        def weight(k, n):
            pw, w = make_weight((g.standard_normal((k, n)) / np.sqrt(k)).astype(H1), quant)
            return pw, w.astype(np.float64)

        def param(v):
            v = np.asarray(v, np.float32)
            return dev(v), v
        self.w_in, self.w_out = weight(WIDTH, ROW), weight(VN, WIDTH)
        self.taps, self.bias = param(g.standard_normal((MIX, TAPS)) / 2), param(g.standard_normal(MIX))
        self.A, self.dt_bias = param(-np.exp(g.uniform(0, 2.5, HEADS))), param(g.standard_normal(HEADS) - 3)
        self.ahead, self.heads, self.behind, self.after, self.channels = (param(1 + 0.3 * g.standard_normal(n)) for n in (WIDTH, VN, WIDTH, WIDTH, WIDTH))
        self.p = fr.Delta(self.A[0].ptr, self.dt_bias[0].ptr, HEADS, KEY_HEADS, DK, DV, DK ** -0.5, EPS, 1, 1)
        self.first = fr.BlockNorm(None, None, self.ahead[0].ptr, None, None, WIDTH, 0, 1, 0, 1.0, EPS)
        self.last = fr.BlockNorm(self.behind[0].ptr, None, self.after[0].ptr, None, self.channels[0].ptr, WIDTH, 1, 1, 0, 0.5, EPS)
        self.conv_state, self.S = dev(np.zeros((seqs, TAPS - 1, MIX), H1)), dev(np.zeros((seqs, HEADS, DK, DV), np.float32))

    def buffers(self, rows, seqs):
        self.a, self.row, self.mix, self.y, self.gated, self.o, self.next = (DevBuf.empty((rows, n), H1) for n in (WIDTH, ROW, MIX, VN, VN, WIDTH, WIDTH))
        self.x = DevBuf.empty((rows, WIDTH), np.float32)
        need = [L().frhip_linear_workspace_bytes(rows, w[0].ref) for w in (self.w_in, self.w_out)]
        self.ws = DevBuf(max(need + [L().frhip_delta_workspace_bytes(C.byref(self.p), seqs, rows), 256]))

    def linear(self, x, ldx, w, y, rows, stream):
        fr.check(L().frhip_linear(x, ldx, w[0].ref, None, 0, None, 0, y, w[0].N, rows, fr.F16, self.ws.ptr, stream), "linear")

    def run(self, rows, starts, stream=None):
        """`starts`: prompts; None: a token of each sequence.  The stream x is taken on in place"""
        x, row, mix = self.x.ptr, self.row.ptr, self.mix.ptr
        fr.check(L().frhip_norm_residual(C.byref(self.first), rows, x, WIDTH, None, 0, None, 0, None, 0, fr.F32, self.a.ptr, WIDTH, fr.F16, stream))
        self.linear(self.a.ptr, WIDTH, self.w_in, row, rows, stream)
        conv = (MIX, TAPS, row, ROW, self.taps[0].ptr, self.bias[0].ptr, 4, self.conv_state.ptr, self.conv_state.ptr, mix, MIX, fr.F16, stream)
        rule = (mix, MIX, mix + 2 * KN, MIX, mix + 4 * KN, MIX, row + 2 * (MIX + VN), ROW, row + 2 * (MIX + VN + HEADS), ROW, self.S.ptr, self.S.ptr, self.y.ptr,
                VN, fr.F16)
        if starts is None:
            fr.check(L().frhip_conv_one(rows, *conv), "conv")
            fr.check(L().frhip_delta_one(C.byref(self.p), rows, *rule, stream), "delta")
        else:
            n, at = len(starts) - 1, (C.c_int32 * len(starts))(*starts)
            fr.check(L().frhip_conv_seq(n, at, *conv), "conv")
            fr.check(L().frhip_delta_seq(C.byref(self.p), n, at, *rule, self.ws.ptr, stream), "delta")
        fr.check(L().frhip_norm_gate(rows, HEADS, DV, 1, self.heads[0].ptr, None, EPS, self.y.ptr, VN, row + 2 * MIX, ROW, 4, self.gated.ptr, VN, fr.F16, stream))
        self.linear(self.gated.ptr, VN, self.w_out, self.o.ptr, rows, stream)
        fr.check(L().frhip_norm_residual(C.byref(self.last), rows, x, WIDTH, self.o.ptr, WIDTH, None, 0, x, WIDTH, fr.F32, self.next.ptr, WIDTH, fr.F16, stream))

    def check(self, x, parts, conv0, S0):
        """`parts`: the rows of each sequence; conv0, S0: the states ahead"""
        a, row, mix, y, gated, o, nxt = (b.numpy().astype(np.float64) for b in (self.a, self.row, self.mix, self.y, self.gated, self.o, self.next))

        def close(got, want, tol, t=H1):
            assert (np.abs(got - want) <= tol + 2.0 ** -10 * tol + half_step(t, want)).all()

        def product(got, a, w):
            _, tol = linear64(a @ w, "none")
            close(got, a @ w, tol((w.shape[0] / 32 + 40) * U * (np.abs(a) @ np.abs(w))))

        def norm(v, err, w):
            return norm64(v, err, "rms", w.astype(np.float64), None)
        x = x.astype(np.float64)
        close(a, *norm(x, np.zeros_like(x), self.ahead[1]))
        product(row, a, self.w_in[1])
        product(o, gated, self.w_out[1])
        conv1, S1 = self.conv_state.numpy(), self.S.numpy()
        for i, r in enumerate(parts):
            want, tol, left = conv64(row[r, :MIX], self.taps[1], self.bias[1], conv0[i], True)
            close(mix[r], want, tol)
            assert np.array_equal(conv1[i], left.astype(H1))
            for h in range(HEADS):
                kh = h // (HEADS // KEY_HEADS)
                hp = dict(A=self.A[1][h], bias=self.dt_bias[1][h], softplus=1, sigmoid=1, eps=np.float64(np.float32(EPS)), scale=np.float64(np.float32(DK ** -0.5)))
                want, tol, S, stol = either(mix[r, kh * DK:(kh + 1) * DK], mix[r, KN + kh * DK:KN + (kh + 1) * DK], mix[r, 2 * KN + h * DV:2 * KN + (h + 1) * DV],
                                            row[r, MIX + VN + h], row[r, MIX + VN + HEADS + h], hp, S0[i, h])
                close(y[r, h * DV:(h + 1) * DV], want, tol)
                assert (np.abs(S1[i, h] - S) <= stol + 2.0 ** -24 * np.abs(S)).all()
        n = len(y)
        v = y.reshape(n, HEADS, DV)
        want, err = norm(v, np.zeros_like(v), self.heads[1].reshape(HEADS, DV))
        want, err = want.reshape(n, VN), err.reshape(n, VN)
        z, ez = act64(row[:, MIX:MIX + VN], np.zeros((n, VN)), "silu")
        close(gated, want * z, err * np.abs(z) + np.abs(want) * ez + 2 * U * np.abs(want * z))
        want, err = norm(o, np.zeros_like(o), self.behind[1])
        c = self.channels[1].astype(np.float64)
        err = err * np.abs(c) + U * np.abs(want * c)
        h = x + 0.5 * want * c
        err = 0.5 * err + U * np.abs(0.5 * want * c) + U * np.abs(h)
        left = self.x.numpy()
        close(left, h, err, np.float32)
        close(nxt, *norm(h, err, self.after[1]))
        return conv1, S1


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("lens", [[83, 7], [5, 130]])
def test_prompts_then_tokens(quant, lens):
    g = np.random.default_rng(1)
    layer, rows = Layer(quant, 2), sum(lens)
    conv, S = layer.conv_state.numpy(), layer.S.numpy()
    layer.buffers(rows, 2)
    x = g.standard_normal((rows, WIDTH)).astype(np.float32)
    layer.x.upload(x)
    layer.run(rows, [0, lens[0], rows])
    fr.check(L().frhip_device_sync())
    conv, S = layer.check(x, [slice(0, lens[0]), slice(lens[0], rows)], conv, S)
    layer.buffers(2, 2)
    for _ in range(3):
        x = g.standard_normal((2, WIDTH)).astype(np.float32)
        layer.x.upload(x)
        layer.run(2, None)
        fr.check(L().frhip_device_sync())
        conv, S = layer.check(x, [slice(0, 1), slice(1, 2)], conv, S)


@pytest.mark.parametrize("starts", [None, [0, 70, 73]])
def test_captured_layers_replay(starts):
    """A layer as one graph, of tokens or of prompts: every replay takes the states on as an eager call does.  Two graphs that run one behind the other share a
    workspace"""
    g = np.random.default_rng(2)
    seqs, rows = (3, 3) if starts is None else (2, starts[-1])
    eager, graphed = [Layer(False, seqs, s) for s in (0, 1)], [Layer(False, seqs, s) for s in (0, 1)]
    st, graphs = C.c_void_p(), [C.c_void_p() for _ in range(2)]
    fr.check(L().frhip_stream_create(C.byref(st)))
    for a in eager + graphed:
        a.buffers(rows, seqs)
    graphed[1].ws = graphed[0].ws
    for a, graph in zip(graphed, graphs):
        fr.check(L().frhip_graph_begin(st))
        a.run(rows, starts, st)
        fr.check(L().frhip_graph_end(st, C.byref(graph)))
    for _ in range(4):
        v = g.standard_normal((rows, WIDTH)).astype(np.float32)
        for a in eager + graphed:
            a.x.upload(v)
        for graph in graphs:
            fr.check(L().frhip_graph_launch(graph, st))
        for a in eager:
            a.run(rows, starts)
        fr.check(L().frhip_stream_sync(st))
        fr.check(L().frhip_device_sync())
        for e, c in zip(eager, graphed):
            for p, q in ((e.next, c.next), (e.x, c.x), (e.S, c.S), (e.conv_state, c.conv_state)):
                assert np.array_equal(p.numpy(), q.numpy())
    for graph in graphs:
        fr.check(L().frhip_graph_destroy(graph))
    fr.check(L().frhip_stream_destroy(st))


def test_two_streams_at_once():
    """Two layers' prompts on streams and workspaces of their own give what each gives alone"""
    g = np.random.default_rng(3)
    x = g.standard_normal((400, WIDTH)).astype(np.float32)
    alone, layers, streams = Layer(True, 2), [Layer(True, 2) for _ in range(2)], [C.c_void_p() for _ in range(2)]
    for a in [alone] + layers:
        a.buffers(400, 2)
    alone.x.upload(x)
    alone.run(400, [0, 330, 400])
    fr.check(L().frhip_device_sync())
    for s in streams:
        fr.check(L().frhip_stream_create(C.byref(s)))
    for _ in range(3):
        for a in layers:
            a.x.upload(x)
            a.conv_state.upload(np.zeros((2, TAPS - 1, MIX), H1))
            a.S.upload(np.zeros((2, HEADS, DK, DV), np.float32))
        for a, s in zip(layers, streams):
            a.run(400, [0, 330, 400], s)
        fr.check(L().frhip_device_sync())
        for a in layers:
            for p, q in ((alone.next, a.next), (alone.x, a.x), (alone.S, a.S), (alone.conv_state, a.conv_state)):
                assert np.array_equal(p.numpy(), q.numpy())
    for s in streams:
        fr.check(L().frhip_stream_destroy(s))
