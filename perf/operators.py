"""The operators of a selective state space layer, as measured cases.

A layer of this kind projects its input, runs a short causal convolution over time, projects the result to a step width
and two vectors per token, runs a scan whose decay depends on the input, and projects back onto the residual stream.
Its operators, each for prompts and for single tokens:

  linear  y = residual + act(x W + bias), x the rows of a wider buffer where they are one
  conv    y[t] = silu(bias + sum_j w[j] x[t - W + 1 + j]), with the last W - 1 inputs as its state
  scan    h = exp(dt A) h + dt B x;  y = (C . h + D x) silu(z);  dt = softplus(dt_raw + dt_bias)

Sequences of a prompt call lie one behind the other; `lens` lists their lengths.
"""
import importlib
import math

import torch

own = False

# Codes of the activations and types, as the library's header has them
_ACT = {"none": 0, "sigmoid": 2, "relu2": 3, "silu": 4, "gelu": 5, "softplus": 6}
_DT = {"f32": (torch.float32, 0), "f16": (torch.float16, 1)}


def _linear(name, t, k, n, ldx=0, weights="f16", act="none", bias=False, residual=False, out="f16"):
    return {"name": name, "op": "linear", "t": t, "k": k, "n": n, "ldx": ldx or k, "weights": weights, "act": act,
            "bias": bias, "residual": residual, "out": out}


def _conv(name, c, w, dtype="f16", rows=0, lens="", ldx=0):
    return {"name": name, "op": "conv", "c": c, "w": w, "dtype": dtype, "rows": rows, "lens": lens, "ldx": ldx or c}


def _scan(name, d, n, groups=1, dtype="f16", rows=0, lens="", gate=True):
    return {"name": name, "op": "scan", "d": d, "n": n, "groups": groups, "dtype": dtype, "rows": rows, "lens": lens,
            "gate": gate}


def listed():
    return [
        # One token of one conversation, a layer of width 2048: back onto the residual stream.  Weights once from memory.
        _linear("linear-token-out", 1, 4096, 2048, residual=True),
        # A step of 48 conversations served together on uint8 weights.
        _linear("linear-batch48-u8", 48, 2048, 8192, weights="u8", act="silu", bias=True),
        # A prompt's step widths: a short K that is no multiple of 64, a slice of the rows that also hold B and C.
        _linear("linear-prompt-dt", 1000, 160, 5120, ldx=192, act="softplus", bias=True, out="f32"),
        # A long prompt back onto the residual stream of a layer of width 2560: the matrix units' work.
        _linear("linear-prompt-out", 4099, 5120, 2560, residual=True),
        # One token each of seven conversations: a launch and its latency.
        _conv("conv-batch7", 4096, 4, rows=7, ldx=8192),
        # A prompt of 4096 tokens, the convolved half of rows that also hold the gate: copy rate.
        _conv("conv-prompt4096", 4096, 4, lens="4096", ldx=8192),
        # Prompts of several conversations in one call, one of them empty, fp32 activations.
        _conv("conv-ragged-f32", 1536, 3, dtype="f32", lens="513,1,0,77,300,2,129,1024,31"),
        # One token of one conversation: latency.
        _scan("scan-token", 4096, 16, rows=1),
        # One token each of 64 conversations: the states once out and back.
        _scan("scan-batch64", 5120, 16, rows=64),
        # One prompt of 4096 tokens, a layer of width 2048.
        _scan("scan-prompt4096", 4096, 16, lens="4096"),
        # Prompts of several conversations in one call, a narrow layer.
        _scan("scan-ragged", 1536, 16, lens="513,1,0,77,300,2,129,1024,31"),
        # Larger states in two groups, fp32 activations.
        _scan("scan-states64-f32", 1280, 64, groups=2, dtype="f32", lens="700,130"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _lens(rng, total):
    """Lengths that add up to `total`: one sequence, or up to twelve of which some are short or empty."""
    if rng.random() < 0.4:
        return str(total)
    cuts = sorted(rng.randint(0, total) for _ in range(rng.randint(1, 11)))
    return ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [total]))


def draw(rng):
    op = rng.choice(["linear", "conv", "scan"])
    one = rng.random() < 0.35
    if op == "linear":
        t = rng.choice([1, 1, 2, 3]) if one else _log(rng, 4, 4099)
        k, n = 8 * _log(rng, 4, 640), _log(rng, 33, 10240)
        while t * k * n > 4099 * 5120 * 2560:
            n = (n + 1) // 2
        return _linear("", t, k, n, ldx=k + rng.choice([0, 0, 8, 32, 40]), weights=rng.choice(["f16", "f16", "u8"]),
                       act=rng.choice(sorted(_ACT)), bias=rng.random() < 0.7, residual=rng.random() < 0.5,
                       out=rng.choice(["f16", "f16", "f32"]))
    dtype = rng.choice(["f16", "f16", "f32"])
    if op == "conv":
        c = _log(rng, 65, 8192)
        ldx = c + rng.choice([0, 1, 32, c])
        w = rng.choice([2, 3, 4, 4])
        if one:
            return _conv("", c, w, dtype, rows=_log(rng, 1, 256), ldx=ldx)
        return _conv("", c, w, dtype, lens=_lens(rng, min(_log(rng, 1, 4096), 4096 * 4096 // c)), ldx=ldx)
    groups = rng.choice([1, 1, 1, 2, 3])
    d, n = groups * _log(rng, 65, 5120 // groups), rng.choice([1, 5, 8, 16, 16, 16, 24, 32, 64, 128])
    gate = rng.random() < 0.8
    if one:
        rows = min(_log(rng, 1, 128), 64 * 5120 * 16 // (d * n) + 1)
        return _scan("", d, n, groups, dtype, rows=rows, gate=gate)
    total = min(_log(rng, 2, 4096), 4096 * 4096 * 16 // (d * n))
    return _scan("", d, n, groups, dtype, lens=_lens(rng, total), gate=gate)


def _starts(case):
    """Rows at which the sequences begin, and behind the last one; None for single tokens."""
    if case["rows"]:
        return None
    at = [0]
    for n in case["lens"].split(","):
        at.append(at[-1] + int(n))
    return at


class _State:
    pass


def _handle(s):
    """What a program that calls the library keeps: its binding, and the addresses of its buffers."""
    fr = importlib.import_module("faster-rwkv_amd")
    s.fr, s.lib = fr, fr.lib()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = _State()
    s.case = case
    {"linear": _prepare_linear, "conv": _prepare_conv, "scan": _prepare_scan}[case["op"]](s, case, normal, uniform)
    return s


# ---- linear ------------------------------------------------------------------------------------------------------
def _quantised(w):
    """uint8 codes of [N][K] with offsets and ranges of its columns n and rows k (binary16)."""
    my = w.amin(0)
    w = w - my
    mx = w.amin(1)
    w = w - mx[:, None]
    rx = w.amax(1)
    w = w / rx[:, None]
    ry = w.amax(0)
    w = w / ry
    q = torch.clamp(torch.floor(w * 256), 0, 255).to(torch.uint8)
    return q, (mx + 0.5 / 256).half(), rx.half(), my.half(), ry.half()


def _prepare_linear(s, case, normal, uniform):
    t, k, n, ldx = case["t"], case["k"], case["n"], case["ldx"]
    s.rows = normal(t, ldx).half()  # the operator reads its first k columns
    w = normal(n, k) / math.sqrt(k)
    s.u8 = case["weights"] == "u8"
    if s.u8:
        s.w, s.mx, s.rx, s.my, s.ry = _quantised(w)
    else:
        s.w = w.half()
    s.bias = normal(n) * 0.5 if case["bias"] else None
    dtype, code = _DT[case["out"]]
    s.residual = normal(t, n).to(dtype) if case["residual"] else None
    s.act = _ACT[case["act"]]
    s.dtype = dtype
    if own:
        _handle(s)
        s.y = torch.empty(t, n, dtype=dtype, device="cuda")
        ptr = [v.data_ptr() if s.u8 else None for v in ([s.mx, s.rx, s.my, s.ry] if s.u8 else [None] * 4)]
        s.weight = s.fr.Weight(s.w.data_ptr(), ptr[0], ptr[1], ptr[2], ptr[3], k, n, s.fr.U8 if s.u8 else s.fr.F16)
        s.ref = s.fr.C.byref(s.weight)
        need = s.lib.frhip_linear_workspace_bytes(t, s.ref)
        s.workspace = torch.empty(max(need, 256), dtype=torch.uint8, device="cuda")
        s.args = (s.rows.data_ptr(), ldx, s.ref, s.bias.data_ptr() if s.bias is not None else None, s.act,
                  s.residual.data_ptr() if s.residual is not None else None, n, s.y.data_ptr(), n, t, code,
                  s.workspace.data_ptr())


def _weight32(s):
    if not s.u8:
        return s.w.float()
    # binary16, as the library's uint8 weights are defined: one rounding of fma(q, rx / 255 * ry, mx + my)
    c = (s.rx.float() / 255)[:, None] * s.ry.float()
    return (s.w.float() * c + (s.mx.float()[:, None] + s.my.float())).half().float()


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-torch.abs(v)))


def _activate(v, act):
    if act == 2:
        return 1 / (1 + torch.exp(-v))
    if act == 3:
        return torch.clamp(v, min=0) ** 2
    if act == 4:
        return v / (1 + torch.exp(-v))
    if act == 5:
        return 0.5 * v * torch.special.erfc(-v / math.sqrt(2))
    if act == 6:
        return _softplus(v)
    return v


def _run_linear(s):
    if own:
        lib, fr = s.lib, s.fr
        fr.check(lib.frhip_linear(*s.args, torch.cuda.current_stream().cuda_stream))
        return s.y
    v = s.rows[:, :s.w.shape[1]].float() @ _weight32(s).t()
    if s.bias is not None:
        v = v + s.bias
    v = _activate(v, s.act)
    if s.residual is not None:
        v = v + s.residual.float()
    return v.to(s.dtype)


def _exact_linear(s, case):
    if s.u8:
        # each code's weight: the real number q rx ry / 255 + mx + my, in the binary16 that the library's products take
        scale = torch.outer(s.rx.double() / 255, s.ry.double())
        w = (s.w.double() * scale + s.mx.double().unsqueeze(1) + s.my.double().unsqueeze(0)).half().double()
    else:
        w = s.w.double()
    p = torch.mm(s.rows[:, :case["k"]].double(), w.t().contiguous())
    if s.bias is not None:
        p += s.bias.double()
    name = case["act"]
    if name == "sigmoid":
        p = torch.reciprocal(torch.exp(-p) + 1)
    elif name == "relu2":
        p = torch.where(p > 0, p * p, torch.zeros_like(p))
    elif name == "silu":
        p = p * torch.reciprocal(torch.exp(-p) + 1)
    elif name == "gelu":
        p = p * (1 + torch.erf(p * math.sqrt(0.5))) / 2
    elif name == "softplus":
        p = torch.logaddexp(p, torch.zeros_like(p))
    if s.residual is not None:
        p += s.residual.double()
    return p


# ---- conv --------------------------------------------------------------------------------------------------------
def _prepare_conv(s, case, normal, uniform):
    c, w, ldx = case["c"], case["w"], case["ldx"]
    dtype, code = _DT[case["dtype"]]
    s.starts = _starts(case)
    seqs = case["rows"] or len(s.starts) - 1
    total = case["rows"] or s.starts[-1]
    s.buf = normal(total, ldx).to(dtype)  # the operator reads its first c columns
    s.x = s.buf[:, :c]
    s.w = (uniform(c, w) * 2 - 1) / math.sqrt(w)
    s.bias = (uniform(c) * 2 - 1) / math.sqrt(w)
    s.state = normal(seqs, w - 1, c).to(dtype)  # the inputs of the tokens before, oldest first
    s.dtype = dtype
    if own:
        _handle(s)
        s.y, s.state_out = torch.empty(total, c, dtype=dtype, device="cuda"), torch.empty_like(s.state)
        head = (seqs,) if s.starts is None else (seqs, (s.fr.C.c_int32 * len(s.starts))(*s.starts))
        s.args = head + (c, w, s.buf.data_ptr(), ldx, s.w.data_ptr(), s.bias.data_ptr(), _ACT["silu"],
                         s.state.data_ptr(), s.state_out.data_ptr(), s.y.data_ptr(), c, code)
        s.call = s.lib.frhip_conv_one if s.starts is None else s.lib.frhip_conv_seq


def _run_conv(s):
    if own:
        s.fr.check(s.call(*s.args, torch.cuda.current_stream().cuda_stream))
        return s.y, s.state_out
    c, w = s.w.shape
    if s.starts is None:
        past = torch.cat([s.state, s.x[:, None]], 1)  # [rows][w][c]
        v = s.bias + (past.float() * s.w.t()).sum(1)
        return (v / (1 + torch.exp(-v))).to(s.dtype), past[:, 1:].contiguous()
    y, states = [], []
    for i, (a, b) in enumerate(zip(s.starts, s.starts[1:])):
        past = torch.cat([s.state[i], s.x[a:b]])
        v = s.bias.expand(b - a, c)
        for j in range(w):
            v = v + past[j:j + b - a].float() * s.w[:, j]
        y.append((v / (1 + torch.exp(-v))).to(s.dtype))
        states.append(past[b - a:])
    return torch.cat(y), torch.stack(states)


def _exact_conv(s, case):
    c, w = case["c"], case["w"]
    parts = [s.x[i:i + 1] for i in range(case["rows"])] if s.starts is None else [s.x[a:b] for a, b in zip(s.starts, s.starts[1:])]
    out, left = [], []
    for before, x in zip(s.state, parts):
        line = torch.cat([before.double(), x.double()])
        left.append(line[len(line) - (w - 1):])
        windows = line.unfold(0, w, 1) if len(x) else line.new_zeros(0, c, w)  # [t][c][w]
        v = (windows * s.w.double()).sum(2) + s.bias.double()
        out.append(v * torch.reciprocal(torch.exp(-v) + 1))
    return torch.cat(out), torch.stack(left)


# ---- scan --------------------------------------------------------------------------------------------------------
def _prepare_scan(s, case, normal, uniform):
    d, n, groups = case["d"], case["n"], case["groups"]
    dtype, code = _DT[case["dtype"]]
    s.starts = _starts(case)
    seqs = case["rows"] or len(s.starts) - 1
    total = case["rows"] or s.starts[-1]
    s.groups, s.dtype = groups, dtype
    u = normal(total, d)
    s.x = (u / (1 + torch.exp(-u))).to(dtype)
    s.dt = (normal(total, d) * 0.5).to(dtype)
    # one row of the projection that gives both, as a program has it: B, then C
    s.bc = normal(total, 2 * groups * n).to(dtype)
    s.z = normal(total, d).to(dtype) if case["gate"] else None
    s.A = -torch.arange(1, n + 1, device="cuda").float() * torch.exp(0.1 * normal(d, n))
    s.D = 1 + 0.1 * normal(d)
    width = torch.exp(uniform(d) * math.log(100) + math.log(0.001))  # step widths of 0.001 to 0.1 at dt = 0
    s.dt_bias = width + torch.log(-torch.expm1(-width))
    s.state = normal(seqs, d, n) * 0.3
    if own:
        _handle(s)
        fr, C = s.fr, s.fr.C
        s.y, s.state_out = torch.empty(total, d, dtype=dtype, device="cuda"), torch.empty_like(s.state)
        s.params = fr.Ssm(s.A.data_ptr(), s.D.data_ptr(), s.dt_bias.data_ptr(), d, n, groups, 1)
        ref = C.byref(s.params)
        head = (ref, seqs) if s.starts is None else (ref, seqs, (C.c_int32 * len(s.starts))(*s.starts))
        ld = 2 * groups * n
        esize = s.bc.element_size()
        tail = ()
        if s.starts is not None:
            s.workspace = torch.empty(max(s.lib.frhip_ssm_workspace_bytes(ref, seqs, total), 256), dtype=torch.uint8, device="cuda")
            tail = (s.workspace.data_ptr(),)
        s.args = head + (s.x.data_ptr(), d, s.dt.data_ptr(), d, s.bc.data_ptr(), ld, s.bc.data_ptr() + groups * n * esize, ld,
                         s.z.data_ptr() if s.z is not None else None, d, s.state.data_ptr(), s.state_out.data_ptr(),
                         s.y.data_ptr(), d, code) + tail
        s.call = s.lib.frhip_ssm_one if s.starts is None else s.lib.frhip_ssm_seq


def _run_scan(s):
    if own:
        s.fr.check(s.call(*s.args, torch.cuda.current_stream().cuda_stream))
        return s.y, s.state_out
    d, n = s.A.shape
    b, c = (v.reshape(-1, s.groups, n) for v in s.bc.float().chunk(2, 1))
    x, dt = s.x.float(), _softplus(s.dt.float() + s.dt_bias)

    def per_channel(v):  # [t][groups][n] -> [t][d][n]
        return v[:, :, None].expand(-1, -1, d // s.groups, -1).reshape(-1, d, n)

    def output(h, lo, hi):
        v = (h * per_channel(c[lo:hi])).sum(2) + s.D * x[lo:hi]
        if s.z is not None:
            z = s.z[lo:hi].float()
            v = v * (z / (1 + torch.exp(-z)))
        return v.to(s.dtype)

    if s.starts is None:
        h = torch.exp(dt[:, :, None] * s.A) * s.state + (dt * x)[:, :, None] * per_channel(b)
        return output(h, 0, len(x)), h
    y, states = [], []
    for i, (a, e) in enumerate(zip(s.starts, s.starts[1:])):
        h = s.state[i]
        for lo in range(a, e, 128):
            hi = min(lo + 128, e)
            decay = torch.exp(dt[lo:hi, :, None] * s.A)
            hs = (dt[lo:hi] * x[lo:hi])[:, :, None] * per_channel(b[lo:hi])
            for t in range(hi - lo):
                h = hs[t].addcmul_(decay[t], h)
            y.append(output(hs, lo, hi))
            h = h.clone()
        states.append(h)
    return torch.cat(y) if y else torch.empty_like(s.x), torch.stack(states)


def _exact_scan(s, case):
    d, n, groups = case["d"], case["n"], case["groups"]
    width = torch.logaddexp(s.dt.double() + s.dt_bias.double(), torch.zeros((), dtype=torch.float64, device="cuda"))
    A, D, x = s.A.double(), s.D.double(), s.x.double()
    B = s.bc[:, :groups * n].double().view(-1, groups, 1, n)
    C = s.bc[:, groups * n:].double().view(-1, groups, n, 1)
    out = torch.empty_like(x)
    rows = [[i] for i in range(case["rows"])] if s.starts is None else [range(a, b) for a, b in zip(s.starts, s.starts[1:])]
    left = []
    for h, steps in zip(s.state.double(), rows):
        h = h.clone()
        for t in steps:
            h *= torch.exp(width[t].unsqueeze(1) * A)
            h += ((width[t] * x[t]).view(groups, -1, 1) * B[t]).view(d, n)
            out[t] = (h.view(groups, -1, n) @ C[t]).view(d)
        left.append(h)
    out += D * x
    if s.z is not None:
        z = s.z.double()
        out *= z * torch.reciprocal(torch.exp(-z) + 1)
    return out, torch.stack(left)


def run(state):
    return {"linear": _run_linear, "conv": _run_conv, "scan": _run_scan}[state.case["op"]](state)


def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "conv": _exact_conv, "scan": _exact_scan}[case["op"]](s, case)


def work(case):
    if case["op"] == "linear":
        t, k, n = case["t"], case["k"], case["n"]
        size = 2 if case["out"] == "f16" else 4
        weights = n * k * 2 if case["weights"] == "f16" else n * k + 4 * (n + k)
        return {"bytes": t * k * 2 + weights + (4 * n if case["bias"] else 0) + t * n * size * (2 if case["residual"] else 1),
                "flops": 2 * t * k * n + 4 * t * n}
    size = 2 if case["dtype"] == "f16" else 4
    starts = _starts(case)
    total = case["rows"] or starts[-1]
    seqs = case["rows"] or len(starts) - 1
    if case["op"] == "conv":
        c, w = case["c"], case["w"]
        return {"bytes": 2 * total * c * size + 2 * seqs * (w - 1) * c * size + 4 * c * (w + 1), "flops": total * c * (2 * w + 4)}
    d, n = case["d"], case["n"]
    return {"bytes": total * (d * (4 if case["gate"] else 3) + 2 * case["groups"] * n) * size + 8 * seqs * d * n + 4 * d * (n + 2),
            "flops": total * d * (8 * n + 12)}
