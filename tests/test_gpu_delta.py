"""The gated delta rule against its formula in float64, for prompts and single tokens."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from hipref import DevBuf, L, dev, fr
from test_gpu_ssm import GUARD, TYPE, U, half_step, seq_table, softplus64

EPS = 1e-6


def delta64(q, k, v, dt, beta, p, state, chunk):
    """One sequence of one head in float64, and what an evaluation in fp32 may be off by: y, its tolerance before rounding, the state behind and its
    tolerance.

    q, k [t][dk], v [t][dv], dt, beta [t].  `chunk`: the rows that are evaluated together, 1 for token by token.  In a chunk that begins at state S the
    written values are U = T R, R_i = b_i (v_i - a_i0 S^T k_i), T the inverse of 1 + L, L_ij = b_i a_ij k_i . k_j (j < i), with a_ij the decay from row j to
    row i; then y_i = scale (a_i0 S^T q_i + sum_j a_ij (q_i . k_j) U_j) and S' = a S + sum_j a_j k_j U_j^T.
    Every operand is held to 2 U of itself at least (fp32, or a pair of binary16 numbers) and the product of two pairs is short of one term of 2 U, so a
    product of n terms is off by (n + 8) U of their magnitudes.  A decay exp(g) is off by (dd + 4 U) |g| + 4 U, dd what the step width is off by (see
    scan64); a vector's length by (dk / 2 + 4) U.  T, found row by row (or block by block), satisfies a 1 + L that is off by (chunk + 8) U of its
    magnitudes (twice that by blocks), which moves T by |T| |dL| |T|.
    A state that is off by E hands on the error that the recurrence makes of it: the columns of S do not mix, and b k k^T in between moves a
    column's length by max(1, |1 - b k.k|) at most, so errors of a state are carried as the lengths of its columns, e."""
    f = np.float64
    q, k, v = q.astype(f), k.astype(f), v.astype(f)
    n, dk = k.shape
    rate = f(p["A"]) if p["A"] is not None else f(1)
    w = dt.astype(f) + (f(p["bias"]) if p["bias"] is not None else 0)
    width = softplus64(w) if p["softplus"] else w
    g = np.where(width == 0, 0, rate * width) if np.isinf(rate) else rate * width
    dg = ((np.abs(w) + 10) * U if p["softplus"] else U) + 4 * U
    dg = np.where(np.isinf(g), 0, dg * np.abs(g))
    b = 1 / (1 + np.exp(-beta.astype(f))) if p["sigmoid"] else beta.astype(f)
    db = ((np.abs(beta.astype(f)) + 6) if p["sigmoid"] else 1) * U * np.abs(b)
    if p["eps"] >= 0:
        k, q = (m / np.sqrt((m * m).sum(1, keepdims=True) + p["eps"]) for m in (k, q))
    q = q * p["scale"]
    dn = (dk / 2 + 6) * U  # of a vector's length, and of what is multiplied by it
    S, e = state.astype(f), np.zeros(v.shape[1])
    y, tol = np.zeros_like(v), np.zeros_like(v)
    mag = np.abs
    for c0 in range(0, n, chunk):
        r = slice(c0, min(n, c0 + chunk))
        K, Q, V, B, dB = k[r], q[r], v[r], b[r][:, None], db[r][:, None]
        m = len(K)
        gr, dgr = g[r], dg[r]
        low = np.tril(np.ones((m, m)))
        # sums of the rows behind j up to i
        gs = np.array([[gr[j + 1:i + 1].sum() for j in range(m)] for i in range(m)])
        ds = np.array([[dgr[j + 1:i + 1].sum() for j in range(m)] for i in range(m)])
        D = np.where(low > 0, np.exp(np.where(low > 0, gs, 0)), 0)
        dD = D * (ds + 4 * U)
        g0, d0 = np.cumsum(gr), np.cumsum(dgr)
        D0, dD0 = np.exp(g0)[:, None], (np.exp(g0) * (d0 + 4 * U))[:, None]
        gram, ag = K @ K.T, mag(K) @ mag(K).T
        Lo = np.tril(B * D * gram, -1)
        dL = np.tril(mag(B) * (dD * ag + D * ag * ((dk + 8) * U + 2 * dn)) + dB * D * ag, -1)
        T = np.linalg.inv(np.eye(m) + Lo)
        dT = mag(T) @ (dL + 2 * (m + 8) * U * (mag(Lo) + np.eye(m))) @ mag(T) if m > 1 else np.zeros((1, 1))
        lenS = np.sqrt((S * S).sum(0)) + e
        lenK, lenQ = np.sqrt((K * K).sum(1))[:, None], np.sqrt((Q * Q).sum(1))[:, None]
        KS, aKS = K @ S, mag(K) @ mag(S)
        R = B * (V - D0 * KS)
        dR = mag(B) * (D0 * aKS * ((dk + 8) * U + dn) + dD0 * aKS + 2 * U * (mag(V) + D0 * aKS)) + (dB + 2 * U * mag(B)) * (mag(V) + D0 * aKS)
        Uv = T @ R
        dU = mag(T) @ dR + dT @ mag(R) + (m + 8) * U * (mag(T) @ mag(R))
        # what the error of S in front makes of the values: the recurrence's own, within the lengths below
        kk = (K * K).sum(1)
        grow = np.array([max(1.0, abs(1 - B[i, 0] * kk[i])) for i in range(m)])
        carried = e[None, :] * np.cumprod(np.exp(gr) * grow)[:, None]  # of the state behind row i
        A = np.tril(D * (Q @ K.T))
        dA = np.tril(dD * (mag(Q) @ mag(K).T) + D * (mag(Q) @ mag(K).T) * ((dk + 8) * U + 2 * dn))
        aA = mag(A) + dA
        y[r] = D0 * (Q @ S) + A @ Uv
        aQS = mag(Q) @ mag(S)
        # A times T times R may be evaluated as (A T) R
        tol[r] = (lenQ * carried + D0 * aQS * ((dk + 8) * U + dn) + dD0 * aQS + aA @ dU + dA @ mag(Uv) + 2 * (m + 8) * U * (aA @ (mag(T) @ mag(R)))
                  + 4 * U * (D0 * aQS + aA @ mag(Uv)))
        back, dback = D[-1][:, None], dD[-1][:, None]
        dS = mag(K * back).T @ dU + (mag(K).T @ ((dback + back * (dn + (m + 8) * U)) * mag(Uv))) + dD0[-1] * mag(S) + 4 * U * mag(D0[-1] * S)
        S = D0[-1] * S + (K * back).T @ Uv
        dS = dS + 2 * U * mag(S)
        e = carried[-1] + np.sqrt((dS * dS).sum(0))
    return y, tol, S, np.broadcast_to(e, S.shape)


def either(*args):
    """The larger of both forms' tolerances: which one a call takes is the library's choice"""
    y, t1, S, s1 = delta64(*args, 1)
    _, t2, _, s2 = delta64(*args, 64)
    return y, np.maximum(t1, t2), S, np.maximum(s1, s2)


def inputs(seed, total, heads, kh, dk, dv, t, pad):
    g = np.random.default_rng(seed)
    silu = lambda m: m / (1 + np.exp(-m))  # noqa: E731
    x = [silu(g.standard_normal((total, kh * dk + pad[0]))).astype(t), silu(g.standard_normal((total, kh * dk + pad[1]))).astype(t),
         silu(g.standard_normal((total, heads * dv + pad[2]))).astype(t), g.standard_normal((total, heads + pad[3])).astype(t),
         g.standard_normal((total, heads + pad[4])).astype(t)]
    return g, x


def delta_case(heads, kh, dk, dv, lens, dtype="f16", one=False, pad=(0, 0, 0, 0, 0, 0), softplus=1, sigmoid=1, norm=True, A=True, bias=True, in_place=False,
               seed=0, change=None, stream=None, check=None, state=None):
    t, code = TYPE[dtype]
    n, total = len(lens), int(sum(lens)) + (0 if one else 2 * GUARD)
    g, x = inputs(seed + heads + dk + dv, total, heads, kh, dk, dv, t, pad)
    if not softplus:
        x[3] = -np.abs(x[3])
    if not sigmoid:
        x[4] = np.clip(np.abs(x[4]), 0, 1.9).astype(t)
    rates = -np.exp(g.uniform(0, 2.5, heads)).astype(np.float32) if softplus else np.full(heads, 0.5, np.float32)
    biases = (g.standard_normal(heads) - 3).astype(np.float32) if softplus else np.zeros(heads, np.float32)
    S0 = (0.3 * g.standard_normal((n, heads, dk, dv))).astype(np.float32) if state is None else state
    if change:
        change(x, rates, biases, S0)
    ldy = heads * dv + pad[5]
    d = [dev(v) for v in x]
    dA, db, ds, dy = dev(rates), dev(biases), dev(S0), dev(np.full((total, ldy), 7, t))
    do = ds if in_place else dev(np.full_like(S0, 9))
    scale, eps = np.float32(1 / np.sqrt(dk)), EPS if norm else -1.0
    p = fr.Delta(dA.ptr if A else None, db.ptr if bias else None, heads, kh, dk, dv, scale, eps, softplus, sigmoid)
    rows = sum(([v.ptr, m.shape[1]] for v, m in zip(d, x)), [])
    args = (*rows, ds.ptr, do.ptr, dy.ptr, ldy, code)
    at, ptr = seq_table(lens)
    if one:
        fr.check(L().frhip_delta_one(C.byref(p), n, *args, stream), "delta_one")
        at = np.arange(n + 1)
    else:
        need = L().frhip_delta_workspace_bytes(C.byref(p), n, int(sum(lens)))
        ws = dev(np.full(need + 64, 0x7b, np.uint8))
        fr.check(L().frhip_delta_seq(C.byref(p), n, ptr, *args, ws.ptr if need else None, stream), "delta_seq")
    fr.check(L().frhip_device_sync())
    if not one:
        assert (ws.numpy()[need:] == 0x7b).all()  # nothing behind the workspace
    y, left = dy.numpy(), do.numpy()
    mine = np.zeros((total, ldy), bool)
    for i in range(n):
        mine[at[i]:at[i + 1], :heads * dv] = True
    assert (y[~mine] == 7).all()
    if check:
        return check(y, left, at, x, S0)
    for i in range(n):
        r = slice(at[i], at[i + 1])
        for h in range(heads):
            kk = h // (heads // kh)
            hp = dict(A=rates[h] if A else None, bias=biases[h] if bias else None, softplus=softplus, sigmoid=sigmoid, eps=eps, scale=np.float64(scale))
            want, tol, S, stol = either(x[0][r, kk * dk:(kk + 1) * dk], x[1][r, kk * dk:(kk + 1) * dk], x[2][r, h * dv:(h + 1) * dv], x[3][r, h], x[4][r, h],
                                        hp, S0[i, h])
            got = y[r, h * dv:(h + 1) * dv].astype(np.float64)
            over = (np.abs(want) + tol >= 65520) & (t == np.float16)  # rounded to binary16 that is infinity
            bad = ~(np.abs(got - want) <= tol + half_step(t, want) + 2.0 ** -10 * tol) & ~(over & (got == np.sign(want) * np.inf))
            assert not bad.any(), ("y", i, h, np.argwhere(bad)[:4], bad.sum(), np.abs(got - want)[bad].max(), tol[bad].max())
            bad = ~(np.abs(left[i, h] - S) <= stol + 2.0 ** -24 * np.abs(S))
            assert not bad.any(), ("state", i, h, np.argwhere(bad)[:4], bad.sum(), np.abs(left[i, h] - S)[bad].max(), stol[bad].max())
    return y, left


SIZES = [(1, 1, 1, 1), (2, 1, 3, 5), (3, 3, 16, 16), (2, 2, 32, 33), (4, 2, 64, 64), (2, 1, 65, 40), (2, 1, 96, 192), (2, 2, 128, 128), (1, 1, 200, 31),
         (2, 1, 256, 256)]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("rows", [1, 3])
def test_single_tokens(size, rows, dtype):
    delta_case(*size, [1] * rows, dtype, one=True)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("lens", [[1], [0, 5, 1], [63, 64, 65], [200]])
def test_prompts(size, lens, dtype):
    delta_case(*size, lens, dtype)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("one", [True, False])
def test_pitches_and_states_in_place(one, dtype):
    lens = [1] * 4 if one else [2, 0, 70, 130]
    delta_case(4, 2, 64, 64, lens, dtype, one, pad=(8, 16, 8, 4, 8, 8), in_place=True)
    delta_case(4, 2, 64, 48, lens, dtype, one, pad=(1, 3, 5, 1, 2, 1), in_place=True, seed=1)
    delta_case(3, 1, 50, 30, lens, dtype, one, pad=(3, 0, 1, 0, 1, 3), seed=2)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("one", [True, False])
def test_without_softplus_sigmoid_norm_or_parameters(one, dtype):
    lens = [1] * 3 if one else [3, 100, 64]
    delta_case(2, 1, 64, 32, lens, dtype, one, softplus=0)
    delta_case(2, 2, 32, 32, lens, dtype, one, softplus=0, A=False, bias=False)
    delta_case(2, 1, 64, 32, lens, dtype, one, sigmoid=0)

    def short(x, rates, biases, S):  # keys as they are, no longer than one
        x[1] *= np.asarray(0.08, x[1].dtype)
    delta_case(2, 1, 64, 32, lens, dtype, one, norm=False, change=short)
    delta_case(2, 2, 64, 32, lens, dtype, one, bias=False, seed=3)


def test_more_prompts_than_a_launch_holds():
    delta_case(1, 1, 16, 16, [i % 4 for i in range(300)], "f16")
    delta_case(2, 1, 16, 16, [(i * 7) % 90 for i in range(140)], "f16")


def test_many_single_tokens():
    delta_case(2, 1, 32, 32, [1] * 700, "f16", one=True)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("n", [40, 150])
def test_keys_that_are_all_alike(n, dtype):
    """Nothing but one key, written at full rate: what a value writes is what the next one takes back"""
    def alike(x, rates, biases, S):
        x[1][:] = x[1][0]
        x[4][:] = 9
        biases[:] = -9
    delta_case(2, 1, 64, 32, [n], dtype, change=alike)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("n", [1, 20, 150])
def test_decays_of_every_size(n, dtype):
    """Rows that forget everything, rows that keep everything, and steep decays beside flat ones in one chunk"""
    def steep(x, rates, biases, S):
        x[3][::3] = 15
        x[3][1::7] = -15
        biases[:] = 0
        rates[0], rates[1] = -np.inf, -1e30
        x[3][:, 2] = 0.01
    delta_case(4, 2, 32, 32, [n], dtype, change=steep)

    def forget(x, rates, biases, S):
        x[3][:] = 0
        x[3][2::5] = -np.inf
        x[3][3::9] = -200
    delta_case(2, 2, 32, 32, [n], dtype, change=forget, softplus=0, A=False, bias=False)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("n", [1, 100])
def test_vectors_of_nothing_and_magnitudes_far_apart(n, dtype):
    def far(x, rates, biases, S):
        x[1][::4] = 0
        x[0][1::4] = 0
        x[2][:, :32] *= np.asarray(1e-3, x[2].dtype)
        x[2][:, 32:] *= np.asarray(3e3, x[2].dtype)
        S[..., 1] *= np.float32(1e9)
        S[..., 3] *= np.float32(1e-9)
        S[..., 5] = 0
    delta_case(2, 1, 64, 32, [n], dtype, change=far)


@pytest.mark.parametrize("one", [True, False])
def test_what_is_not_finite_stays_in_its_head_and_behind_its_token(one):
    """A value in its column, a key, decay or rate in its head, from its token on; a query in its row"""
    heads, dk, dv = 4, 32, 32
    n = 1 if one else 100
    clean = {}
    for name in ("v", "k", "q", "beta", "dt", "state", "inf"):
        at = 0 if one else 40

        def spoil(x, rates, biases, S):
            row = at + (0 if one else GUARD)
            if name == "v":
                x[2][row, dv + 3] = np.nan
            elif name == "inf":
                x[2][row, dv + 3] = np.inf
            elif name == "k":
                x[1][row, dk:2 * dk] = np.nan
            elif name == "q":
                x[0][row, dk + 5] = np.nan
            elif name == "beta":
                x[4][row, 1] = np.nan
            elif name == "dt":
                x[3][row, 1] = np.nan
            else:
                S[0, 1, 4, 3] = np.nan

        def look(y, left, starts, x, S0):
            return y[starts[0]:starts[1]].reshape(n, heads, dv).astype(np.float32), left[0]
        if not clean:
            clean["y"], clean["S"] = delta_case(heads, heads, dk, dv, [n], one=one, check=look)
        y, S = delta_case(heads, heads, dk, dv, [n], one=one, change=spoil, check=look)
        ybad, Sbad = np.zeros(y.shape, bool), np.zeros(S.shape, bool)
        if name in ("v", "inf"):
            ybad[at:, 1, 3] = Sbad[1, :, 3] = True
        elif name == "state":
            ybad[:, 1, 3] = Sbad[1, :, 3] = True
        elif name == "q":
            ybad[at, 1] = True
        else:
            ybad[at:, 1] = Sbad[1] = True
        assert np.array_equal(y[~ybad], clean["y"][~ybad]) and np.array_equal(S[~Sbad], clean["S"][~Sbad]), name
        assert not np.isfinite(y[ybad]).any() or name == "inf", name
        assert not np.isfinite(S[Sbad]).any() or name in ("state", "inf"), name


@pytest.mark.parametrize("n", [3, 150])
def test_results_repeat(n):
    def look(y, left, starts, x, S0):
        return y, left
    a, b = (delta_case(4, 2, 128, 64, [n, 17], check=look) for _ in range(2))
    assert all(np.array_equal(p, q) for p, q in zip(a, b))
