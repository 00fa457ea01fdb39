"""Measured cases of the operators of a recurrent layer: norm, 8-bit product, state space scan.

Three operators, as such a layer uses them one behind the other: the
root-mean-square norm (with the residual's addition, or over heads with a gate;
its output in f32 or in 8 bits with a scale for each row), the matrix product in
8-bit integers with scales for each token and channel, and the selective state
space scan with its short causal convolution, for prompts and for single tokens.
`listed()` names the cases, `draw()` gives more of the same ranges, `prepare()`
makes what a program holds before the call, `run()` is one call (in plain torch
operations, or the library's where `own` is true) and `exact()` the same result
in 64 bits.

A scan's requests have lengths that are spread evenly over their logarithm
between two ends, so that a case's work is known without its seed; which request
has which length goes by the seed.  Every request but each fifth has tokens
behind it.
"""
import math

import torch

own = False

EPS = 1e-6
DELTA, STATE = 0, 1


def listed():
    return [
        # Between two blocks, one token: latency alone.
        {"name": "norm_token", "kind": "norm", "rows": 1, "cols": 2048, "group": 2048, "res": True, "gate": False, "i8": False},
        # Between two blocks of a long prompt, for a product in 8 bits.
        {"name": "norm_prompt_i8", "kind": "norm", "rows": 2048, "cols": 2048, "group": 2048, "res": True, "gate": False, "i8": True},
        # The mixer's output of a long prompt: heads of 128 normed apart, gated.
        {"name": "norm_heads", "kind": "norm", "rows": 2048, "cols": 4096, "group": 128, "res": False, "gate": True, "i8": False},
        # The mixer's output projection of one token.
        {"name": "mm_token", "kind": "mm", "T": 1, "rows": 2048, "cols": 4096},
        # The mixer's input projections (8192 channels and 4096 gates) of eight slots.
        {"name": "mm_slots8", "kind": "mm", "T": 8, "rows": 12288, "cols": 2048},
        # The same for a prompt's chunk of the reference's size, and for a long prompt.
        {"name": "mm_chunk", "kind": "mm", "T": 256, "rows": 12288, "cols": 2048},
        {"name": "mm_prompt", "kind": "mm", "T": 2048, "rows": 12288, "cols": 2048},
        # Sizes that fill no tile.
        {"name": "mm_odd", "kind": "mm", "T": 333, "rows": 1111, "cols": 2064},
        # One token of one chat.
        {"name": "scan_token", "kind": "scan", "mode": DELTA, "n": 1, "lo": 1, "hi": 1, "idle": 0, "pad": 0, "kh": 16, "vh": 32,
         "kd": 128, "vd": 128, "taps": 4, "skip": False},
        # A large batch of single tokens, some requests idle, rows behind the last.
        {"name": "scan_slots64", "kind": "scan", "mode": DELTA, "n": 64, "lo": 1, "hi": 1, "idle": 6, "pad": 6, "kh": 16, "vh": 32,
         "kd": 128, "vd": 128, "taps": 4, "skip": False},
        # A long prompt.
        {"name": "scan_prompt", "kind": "scan", "mode": DELTA, "n": 1, "lo": 2048, "hi": 2048, "idle": 0, "pad": 0, "kh": 16,
         "vh": 32, "kd": 128, "vd": 128, "taps": 4, "skip": False},
        # Ragged prompts through the form without the correction, many heads on one group of keys.
        {"name": "scan_ragged_state", "kind": "scan", "mode": STATE, "n": 5, "lo": 37, "hi": 700, "idle": 1, "pad": 11, "kh": 1,
         "vh": 24, "kd": 128, "vd": 64, "taps": 4, "skip": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "mm", "mm", "scan", "scan", "scan"])
    if kind == "norm":
        group = rng.choice([0, 0, 0, 64, 128, 256])
        cols = group * rng.randint(1, 32) if group else 4 * _log_int(rng, 16, 2048)
        return {"kind": kind, "rows": _log_int(rng, 1, 2048), "cols": cols, "group": group or cols, "res": rng.random() < 0.6,
                "gate": rng.random() < 0.4, "i8": rng.random() < 0.5}
    if kind == "mm":
        return {"kind": kind, "T": _log_int(rng, 1, 2048), "rows": _log_int(rng, 64, 12288), "cols": 16 * _log_int(rng, 16, 256)}
    heads = rng.choice([(16, 32, 128, 128)] * 3 + [(4, 4, 64, 128), (1, 40, 128, 64), (2, 12, 64, 64), (8, 8, 128, 128)])
    c = {"kind": kind, "mode": rng.choice([DELTA, DELTA, STATE]), "n": 1, "lo": 1, "hi": 1, "idle": 0, "pad": rng.choice([0, rng.randint(1, 20)]),
         "kh": heads[0], "vh": heads[1], "kd": heads[2], "vd": heads[3], "taps": rng.choice([4, 4, 3, 2]), "skip": rng.random() < 0.5}
    form = rng.choice(["token", "draft", "prompt", "prompt"])
    c["n"] = _log_int(rng, 1, 64) if form != "prompt" else rng.randint(1, 6)
    if form == "draft":
        c["hi"] = rng.randint(2, 8)
    if form == "prompt":
        c["hi"] = _log_int(rng, 20, 2048 // c["n"])
        c["lo"] = max(1, int(c["hi"] * rng.uniform(0.05, 1)))
    c["idle"] = rng.randint(0, c["n"] // 3)
    return c


# ---- sizes -------------------------------------------------------------------
def _spread(n, lo, hi):
    """n lengths from lo to hi, even over their logarithm."""
    a, b = math.log(lo), math.log(hi)
    return [int(round(math.exp(a + (b - a) * i / max(1, n - 1)))) for i in range(n)]


def _new(case):
    """New tokens of each request; the first ones are idle."""
    return [0 if i < case["idle"] else v for i, v in enumerate(_spread(case["n"], case["lo"], case["hi"]))]


def _channels(case):
    return 2 * case["kh"] * case["kd"] + case["vh"] * case["vd"]


def work(case):
    """Inputs read once, outputs written once."""
    k = case["kind"]
    if k == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (4 + 8 * case["res"] + 4 * case["gate"] + (1 if case["i8"] else 4)) + 4 * case["group"] +
                4 * case["rows"] * case["i8"], "flops": 6.0 * n}
    if k == "mm":
        T, N, K = case["T"], case["rows"], case["cols"]
        return {"bytes": T * K + N * K + 4 * (T * N + T + N), "flops": 2.0 * T * N * K}
    new, C = [m for m in _new(case) if m], _channels(case)
    T, live = sum(new), len(new)
    out = case["vh"] * case["vd"]
    delta = case["mode"] == DELTA
    state = 4 * case["vh"] * case["kd"] * case["vd"]
    return {"bytes": 4 * T * (C + out + (2 if delta else 1) * case["vh"]) + live * 2 * state +
            4 * C * (sum(case["taps"] - 1 + min(m, case["taps"]) for m in new) + case["taps"] + 1),
            "flops": T * (2.0 * C * case["taps"] + (8.0 if delta else 5.0) * case["vh"] * case["kd"] * case["vd"])}


# ---- state -------------------------------------------------------------------
class _State:
    pass


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _uniform(g, lo, hi, *shape):
    return lo + (hi - lo) * torch.rand(*shape, device="cuda", generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_norm(s, case, g):
    T, D = case["rows"], case["cols"]
    # a few channels stand far above the others, as a residual stream's do
    tall = 1 + 12 * (torch.rand(D, device="cuda", generator=g) < 0.004)
    s.x = _normal(g, T, D) * tall
    s.res = _normal(g, T, D) * tall if case["res"] else None
    s.gate = 2 * _normal(g, T, D) if case["gate"] else None
    s.group, s.weight = case["group"], 1 + 0.2 * _normal(g, case["group"])
    s.y = s.q = s.q_scale = s.values = None
    if case["i8"]:
        s.q, s.q_scale = torch.zeros(T, D, dtype=torch.int8, device="cuda"), torch.zeros(T, device="cuda")
        s.values = torch.zeros(T, D, dtype=torch.float16, device="cuda")
    else:
        s.y = torch.zeros(T, D, device="cuda")


def _prepare_mm(s, case, g):
    T, N, K = case["T"], case["rows"], case["cols"]

    def eights(rows):                                      # rows in 8 bits, the largest of each at 127
        v = _normal(g, rows, K)
        top = v.abs().amax(dim=1, keepdim=True)
        return torch.round(v * (127 / top)).to(torch.int8), (top / 127).flatten()
    s.xq, s.xs = eights(T)
    s.wq, s.ws = eights(N)
    s.y = torch.zeros(T, N, device="cuda")


def _prepare_scan(s, case, g):
    n, kh, vh, kd, vd, taps = (case[k] for k in ("n", "kh", "vh", "kd", "vd", "taps"))
    host = torch.Generator().manual_seed(g.initial_seed())
    order = torch.randperm(n, generator=host).tolist()
    new = _new(case)
    s.new = [new[i] for i in order]
    far = torch.randint(1, 5000, (n,), generator=host).tolist()
    s.behind = [0 if i % 5 == 4 else far[i] for i in range(n)]     # tokens of each request before these
    T, C = sum(s.new), _channels(case)
    s.mode, s.kh, s.vh, s.kd, s.vd, s.taps, s.C = case["mode"], kh, vh, kd, vd, taps, C
    s.scale = kd ** -0.5 if s.mode == DELTA else 1.0
    rows = T + case["pad"]
    s.x = _normal(g, rows, C)
    s.a, s.b = 1.5 * _normal(g, rows, vh), _normal(g, rows, vh)
    s.conv_w, s.conv_b = _normal(g, C, taps) / math.sqrt(taps), 0.1 * _normal(g, C)
    s.a_coef = -torch.exp(_uniform(g, 0, math.log(16), vh))
    s.dt_bias = torch.log(torch.expm1(torch.exp(_uniform(g, math.log(0.001), math.log(0.1), vh))))
    s.skip = 1 + 0.1 * _normal(g, vh) if case["skip"] else None
    s.conv, s.state = _normal(g, n, taps, C), 0.3 * _normal(g, n, vh, vd, kd)
    s.first = _ints([sum(s.new[:i]) for i in range(n + 1)])
    s.row_pos = _ints([b + i for m, b in zip(s.new, s.behind) for i in range(m)] + [-1] * case["pad"])
    s.out = torch.zeros(rows, vh, vd, device="cuda")
    s.rows, s.most = rows, max(s.new)
    # of each row: its request, and the row or the conv entry of each tap (entries behind the rows, zeros at the end)
    at, req = [], []
    for r, (m, b) in enumerate(zip(s.new, s.behind)):
        for i in range(m):
            req.append(r)
            for j in range(taps):
                d = i - (taps - 1) + j
                at.append(len(req) - 1 - i + d if d >= 0 else T + r * taps + (b + d) % taps if b + d >= 0 else T + n * taps)
    s.tap = torch.tensor(at, device="cuda").reshape(T, taps)
    s.valid = T
    # the requests of each step of the recurrence, and their rows
    f = s.first.tolist()
    steps = [[r for r in range(n) if s.new[r] > i] for i in range(s.most)]
    s.steps = [(torch.tensor(q, device="cuda"), torch.tensor([f[r] + i for r in q], device="cuda")) for i, q in enumerate(steps)] if n > 1 \
        else [(slice(0, 1), slice(i, i + 1)) for i in range(s.most)]
    s.fresh = torch.tensor([m > 0 and not b for m, b in zip(s.new, s.behind)], device="cuda")
    # the conv entries that the step leaves: the last rows of each request
    keep = [(r, (s.behind[r] + i) % taps, f[r] + i) for r in range(n) for i in range(max(0, s.new[r] - taps), s.new[r])]
    s.keep_req, s.keep_at, s.keep_row = (torch.tensor([k[i] for k in keep], device="cuda") for i in range(3))


def prepare(case, seed):
    s = _State()
    s.kind = case["kind"]
    g = _gen(seed)
    {"norm": _prepare_norm, "mm": _prepare_mm, "scan": _prepare_scan}[s.kind](s, case, g)
    if own:
        _bind(s)
    return s


def _bind(s):
    """The argument structures of the library's calls; the product's weights in its order."""
    import ctypes as C

    import roaster_amd as R
    L = R.lib()
    R.check(L.roaster_init(), "init")
    if s.kind == "norm":
        T, D = s.x.shape
        a = R.RoasterNorm(T, D, s.group, R.ptr(s.x), D, R.ptr(s.res), D, R.ptr(s.weight), R.ptr(s.gate), D, EPS, R.ptr(s.y), D,
                          R.ptr(s.q), D, R.ptr(s.q_scale))
        s.call, s.args, s.keep = L.roaster_norm, (C.byref(a),), (a,)
        s.stream = torch.cuda.ExternalStream(L.roaster_stream())
        return
    if s.kind == "mm":
        (N, K), T = s.wq.shape, s.xq.shape[0]
        s.packed = torch.empty(L.roaster_i8_bytes(N, K), dtype=torch.uint8, device="cuda")
        w = R.RoasterI8(R.ptr(s.packed), R.ptr(s.ws), N, K)
        torch.cuda.synchronize()
        R.check(L.roaster_i8_pack(R.ptr(s.wq), R.I8_FROM_I8, C.byref(w)), "i8_pack")
        a = R.RoasterMatmulI8(T, R.ptr(s.xq), K, R.ptr(s.xs), R.ptr(s.y), N)
        s.call, s.args, s.keep = L.roaster_matmul_i8, (C.byref(a), C.byref(w)), (a, w)
        return
    st = R.RoasterSsmState(len(s.new), s.kh, s.vh, s.kd, s.vd, s.taps, R.ptr(s.conv), R.ptr(s.state))
    s.work = torch.empty(L.roaster_ssm_ws_bytes(s.rows, s.most, C.byref(st)), dtype=torch.uint8, device="cuda")
    a = R.RoasterSsmScan(s.rows, s.most, s.mode, R.ptr(s.x), s.C, R.ptr(s.a), s.vh, R.ptr(s.b) if s.mode == DELTA else None, s.vh,
                         R.ptr(s.conv_w), R.ptr(s.conv_b), R.ptr(s.a_coef), R.ptr(s.dt_bias), R.ptr(s.skip), s.scale, EPS,
                         R.ptr(s.first), R.ptr(s.row_pos), R.ptr(s.out), s.vh * s.vd, R.ptr(s.work), s.work.numel())
    s.call, s.args, s.keep = L.roaster_ssm_scan, (C.byref(a), C.byref(st)), (a, st)


# ---- the operators, plainly ----------------------------------------------------
def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _norm(s):
    x = s.x
    if s.res is not None:
        s.res += s.x
        x = s.res
    v = x.view(x.shape[0], -1, s.group)
    y = (v * torch.rsqrt((v * v).mean(dim=-1, keepdim=True) + EPS) * s.weight).view(x.shape)
    if s.gate is not None:
        y = y * (s.gate * _sigmoid(s.gate))
    if s.q is None:
        s.y.copy_(y)
        return
    top = y.abs().amax(dim=1, keepdim=True)
    s.q_scale.copy_((top / 127).flatten())
    s.q.copy_(torch.round(y * (127 / top)))


def _mm(s):
    s.y.copy_((s.xq.float() @ s.wq.float().T) * s.xs[:, None] * s.ws)


def _scan(s):
    """Token by token, the requests' side by side."""
    T, n, C = s.valid, len(s.new), s.C
    rows = torch.cat([s.x[:T], s.conv.view(-1, C), torch.zeros(1, C, device=s.x.device)])
    c = s.conv_b.expand(T, C)
    for j in range(s.taps):
        c = c + rows[s.tap[:, j]] * s.conv_w[:, j]
    c = c * _sigmoid(c)
    nk = s.kh * s.kd
    q, k, v = c[:, :nk].view(T, s.kh, s.kd), c[:, nk:2 * nk].view(T, s.kh, s.kd), c[:, 2 * nk:].view(T, s.vh, s.vd, 1)
    a = s.a[:T] + s.dt_bias
    dt = a.clamp(min=0) + torch.log1p(torch.exp(-a.abs()))
    decay = torch.exp(s.a_coef * dt)[..., None, None]
    if s.mode == DELTA:
        q, k = (z * torch.rsqrt((z * z).sum(dim=-1, keepdim=True) + EPS) for z in (q, k))
        gain = _sigmoid(s.b[:T])[..., None, None]
    else:
        gain = dt[..., None, None]
    # [T, vh, kd, 1] and [T, vh, 1, kd]
    q, k = ((z.repeat_interleave(s.vh // s.kh, dim=1)) for z in (q * s.scale, k))
    q, kc, kr = q[..., None], k[..., None], k[:, :, None, :]
    S = s.state.masked_fill(s.fresh.view(n, 1, 1, 1), 0)
    out = torch.empty(T, s.vh, s.vd, 1, device=s.x.device)
    for req, at in s.steps:                                # S [n, vh, vd, kd]
        P = S[req] * decay[at]
        d = v[at] - P @ kc[at] if s.mode == DELTA else v[at]
        P = P + (gain[at] * d) * kr[at]
        out[at] = P @ q[at]
        S[req] = P
    s.out[:T] = out[..., 0] if s.skip is None else out[..., 0] + s.skip[:, None] * v[..., 0]
    s.state.copy_(S)
    s.conv[s.keep_req, s.keep_at] = s.x[s.keep_row]


def _outputs(s):
    if s.kind == "norm":
        return [v for v in (s.res, s.y, s.values, s.q_scale) if v is not None]
    return s.y if s.kind == "mm" else [s.out, s.conv, s.state]


def run(s):
    if own:
        rc = s.call(*s.args)
        if rc:
            raise RuntimeError("call failed (%d)" % rc)
        if s.kind == "norm" and s.q is not None:           # what the 8 bits stand for
            with torch.cuda.stream(s.stream):
                torch.mul(s.q, s.q_scale[:, None], out=s.values)
        return _outputs(s)
    {"norm": _norm, "mm": _mm, "scan": _scan}[s.kind](s)
    if s.kind == "norm" and s.q is not None:
        torch.mul(s.q, s.q_scale[:, None], out=s.values)
    return _outputs(s)


# ---- the same in 64 bits -----------------------------------------------------
def _exact_norm(s):
    x = s.x.double() if s.res is None else s.x.double() + s.res.double()
    h = x.reshape(-1, s.group)
    y = h / torch.sqrt(torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / s.group + EPS) * s.weight.double()
    y = y.view(x.shape)
    if s.gate is not None:
        y = y * torch.nn.functional.silu(s.gate.double())
    got = [] if s.res is None else [x]
    if s.q is None:
        return got + [y]
    step = y.abs().max(dim=1).values / 127
    return got + [(y / step[:, None]).round() * step[:, None], step]


def _exact_mm(s):
    """By blocks of channels, scales first."""
    x = s.xq.double() * s.xs.double()[:, None]
    return torch.cat([x @ (w.double() * sc.double()[:, None]).T.contiguous() for w, sc in zip(s.wq.split(2048), s.ws.split(2048))], dim=1)


def _exact_scan(s):
    """Request by request in pieces of 32 tokens: within a piece the corrections solve a triangular system."""
    F = torch.nn.functional
    out, conv, state = s.out.double(), s.conv.double(), s.state.double()
    f, rep, nk = s.first.tolist(), s.vh // s.kh, s.kh * s.kd
    for r, m in enumerate(s.new):
        if not m:
            continue
        b, x = s.behind[r], s.x[f[r]:f[r] + m].double()
        past = torch.stack([conv[r, (b - i) % s.taps] if b >= i else torch.zeros_like(x[0]) for i in range(s.taps - 1, 0, -1)])
        c = F.silu(F.conv1d(torch.cat([past, x]).T[None], s.conv_w.double()[:, None], s.conv_b.double(), groups=s.C)[0].T)
        for i in range(max(0, m - s.taps), m):
            conv[r, (b + i) % s.taps] = x[i]
        q, k, v = c[:, :nk].reshape(m, s.kh, s.kd), c[:, nk:2 * nk].reshape(m, s.kh, s.kd), c[:, 2 * nk:].reshape(m, s.vh, s.vd)
        dt = F.softplus(s.a[f[r]:f[r] + m].double() + s.dt_bias.double(), threshold=100)
        log, gain = dt * s.a_coef.double(), dt
        if s.mode == DELTA:
            q, k = (z / torch.sqrt(z.pow(2).sum(-1, keepdim=True) + EPS) for z in (q, k))
            gain = torch.sigmoid(s.b[f[r]:f[r] + m].double())
        q, k = (z.repeat_interleave(rep, 1).transpose(0, 1).contiguous() for z in (q * s.scale, k))     # [vh, m, kd]
        vt, log, gain = v.transpose(0, 1), log.T, gain.T
        S = state[r].transpose(1, 2).contiguous() if b else torch.zeros(s.vh, s.kd, s.vd, dtype=torch.float64, device="cuda")
        for i in range(0, m, 32):
            Q, K, V, G, B = q[:, i:i + 32], k[:, i:i + 32], vt[:, i:i + 32], log[:, i:i + 32].cumsum(1), gain[:, i:i + 32, None]
            w = K.shape[1]
            late = torch.ones(w, w, dtype=torch.bool, device="cuda").triu(1)
            D = (G[:, :, None] - G[:, None, :]).masked_fill(late, -math.inf).exp()
            U = B * V
            if s.mode == DELTA:
                A = (B * (K @ K.transpose(1, 2).contiguous()) * D).tril(-1) + torch.eye(w, dtype=torch.float64, device="cuda")
                U = torch.linalg.solve_triangular(A, U - B * G.exp()[..., None] * (K @ S), upper=False, unitriangular=True)
            out[f[r] + i:f[r] + i + w] = (G.exp()[..., None] * (Q @ S) + ((Q @ K.transpose(1, 2).contiguous()) * D) @ U).transpose(0, 1)
            S = G[:, -1:, None].exp() * S + (K * (G[:, -1:] - G).exp()[..., None]).transpose(1, 2).contiguous() @ U
        if s.skip is not None:
            out[f[r]:f[r] + m] += s.skip.double()[:, None] * v
        state[r] = S.transpose(1, 2)
    return [out, conv, state]


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "mm": _exact_mm, "scan": _exact_scan}[s.kind](s)
