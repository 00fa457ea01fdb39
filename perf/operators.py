"""Measured cases of the attention operators over a paged key/value cache.

Three operators, as one serving step uses them: the plan (block tables, row
positions and cache slots from the requests' lengths), the query/key norms with
the position rotation and the store into the cache, and attention over the
cached pages.  `listed()` names the cases, `draw()` gives more of the same
ranges, `prepare()` makes what a program holds before the call, `run()` is one
call (in plain torch operations, or the library's where `own` is true) and
`exact()` the same result in 64 bits.

A cache page holds `page` tokens of every key/value head:
[n_pages][kv_heads][page][dim], keys and values apart.  Requests' lengths are
spread evenly over their logarithm between two ends, so that a case's work is
known without its seed; which request has which length goes by the seed.
"""
import math

import torch

own = False

EPS = 1e-6
THETA = 1e7
F32, F16 = 0, 1
DTYPE = {F32: torch.float32, F16: torch.float16}


def listed():
    return [
        # One decode step of the eight slots that a server runs together.
        {"name": "plan_slots8", "kind": "plan", "n": 8, "lo": 40, "hi": 6000, "page": 64, "chunk": 1, "pad": 0},
        # A large server's step: most requests add one token, some a prompt chunk, some have ended; padded for a graph.
        {"name": "plan_mixed_512", "kind": "plan", "n": 512, "lo": 1, "hi": 9000, "page": 16, "chunk": 256, "pad": 300},
        # The attention layer's projections of one token.
        {"name": "rope_token", "kind": "rope", "rows": 1, "pad": 0, "heads": 16, "kv": 2, "dim": 256, "rot": 64,
         "adjacent": False, "norm": True, "far": 5000, "page": 64, "type": F16},
        # Forty-eight requests far into long contexts, the cache in f32 as the reference keeps it.
        {"name": "rope_far_f32", "kind": "rope", "rows": 48, "pad": 0, "heads": 16, "kv": 2, "dim": 256, "rot": 64,
         "adjacent": False, "norm": True, "far": 1000000, "page": 64, "type": F32},
        # A long prompt.
        {"name": "rope_prompt", "kind": "rope", "rows": 2048, "pad": 0, "heads": 16, "kv": 2, "dim": 256, "rot": 64,
         "adjacent": False, "norm": True, "far": 2048, "page": 64, "type": F16},
        # Another model's heads: every query head with its own keys, all of it rotated by neighbours, no norms, padded rows.
        {"name": "rope_odd", "kind": "rope", "rows": 333, "pad": 19, "heads": 8, "kv": 8, "dim": 128, "rot": 128,
         "adjacent": True, "norm": False, "far": 30000, "page": 16, "type": F16},
        # The first tokens of a single chat: latency alone.
        {"name": "attn_chat", "kind": "attn", "n": 1, "each": 1, "idle": 0, "lo": 437, "hi": 437, "heads": 16, "kv": 2,
         "dim": 256, "page": 64, "type": F16, "gate": True, "pad": 0},
        # Eight slots of ragged lengths, two of them idle.
        {"name": "attn_slots", "kind": "attn", "n": 8, "each": 1, "idle": 2, "lo": 100, "hi": 8000, "heads": 16, "kv": 2,
         "dim": 256, "page": 64, "type": F16, "gate": True, "pad": 3},
        # A large batch of ragged lengths.
        {"name": "attn_batch64", "kind": "attn", "n": 64, "each": 1, "idle": 0, "lo": 300, "hi": 16000, "heads": 16,
         "kv": 2, "dim": 256, "page": 16, "type": F16, "gate": True, "pad": 0},
        # One request with a very long context.
        {"name": "attn_long", "kind": "attn", "n": 1, "each": 1, "idle": 0, "lo": 200001, "hi": 200001, "heads": 16,
         "kv": 2, "dim": 256, "page": 256, "type": F16, "gate": False, "pad": 0},
        # An f32 cache and other heads.
        {"name": "attn_f32", "kind": "attn", "n": 12, "each": 1, "idle": 0, "lo": 500, "hi": 5000, "heads": 32, "kv": 8,
         "dim": 128, "page": 32, "type": F32, "gate": False, "pad": 0},
        # A prompt's chunk of the reference's size behind what is cached already.
        {"name": "attn_chunk", "kind": "attn", "n": 1, "each": 256, "idle": 0, "lo": 2304, "hi": 2304, "heads": 16,
         "kv": 2, "dim": 256, "page": 64, "type": F16, "gate": True, "pad": 0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "rope", "attn", "attn", "attn", "attn"])
    page = rng.choice([16, 16, 32, 64, 64, 128, 256])
    if kind == "plan":
        return {"kind": kind, "n": _log_int(rng, 1, 700), "lo": rng.randint(0, 50), "hi": _log_int(rng, 60, 9000),
                "page": page, "chunk": rng.choice([1, 1, rng.randint(2, 256)]), "pad": rng.randint(0, 300)}
    heads, kv, dim = rng.choice([(16, 2, 256)] * 4 + [(32, 8, 128), (8, 8, 128), (20, 4, 64), (7, 1, 128), (16, 1, 64)])
    if kind == "rope":
        return {"kind": kind, "rows": _log_int(rng, 1, 2048), "pad": rng.choice([0, 0, rng.randint(1, 40)]),
                "heads": heads, "kv": kv, "dim": dim, "rot": rng.choice([dim, dim // 2, dim // 4, 64 if dim > 64 else 24]),
                "adjacent": rng.random() < 0.3, "norm": rng.random() < 0.8, "far": _log_int(rng, 3000, 1000000),
                "page": page, "type": rng.choice([F16, F16, F32])}
    c = {"kind": kind, "n": 1, "each": 1, "idle": 0, "lo": 1, "hi": 1, "heads": heads, "kv": kv, "dim": dim, "page": page,
         "type": rng.choice([F16, F16, F16, F32]), "gate": rng.random() < 0.6, "pad": rng.choice([0, 0, rng.randint(1, 9)])}
    form = rng.choice(["decode", "decode", "draft", "chunk"])
    if form == "chunk":                                    # a prompt's rows
        c["n"], c["each"] = rng.choice([(1, rng.randint(17, 256)), (2, rng.randint(17, 128))])
        c["hi"] = c["each"] + _log_int(rng, 1, 3000)
    else:
        c["n"] = _log_int(rng, 1, 64)
        c["each"] = rng.randint(2, 6) if form == "draft" else 1
        most = 200e6 / (c["n"] * 2 * kv * dim * 4)         # tokens a request, by the plain form's f32 copies
        c["hi"] = c["each"] + _log_int(rng, 1, max(2, min(200000, most)))
        c["idle"] = rng.randint(0, c["n"] // 2)
    c["lo"] = max(c["each"], int(c["hi"] * rng.uniform(0.02, 1)))
    return c


# ---- sizes -------------------------------------------------------------------
def _spread(n, lo, hi):
    """n lengths from lo to hi, even over their logarithm."""
    a, b = math.log(lo + 1), math.log(hi + 1)
    return [int(round(math.exp(a + (b - a) * i / max(1, n - 1)))) - 1 for i in range(n)]


def _steps(case):
    """(cached tokens, new tokens) of each request of a plan: one new token, every fifth
    a prompt chunk, every eleventh ended (-1), every thirteenth idle."""
    add = [-1 if i % 11 == 5 else 0 if i % 13 == 7 else case["chunk"] if i % 5 == 3 else 1 for i in range(case["n"])]
    return list(zip(_spread(case["n"], case["lo"], case["hi"]), add))


def _pages(tokens, page):
    return -(-tokens // page)


def _lengths(case):
    """Tokens of each request, its new rows among them; the first ones are idle."""
    return [0 if i < case["idle"] else v for i, v in enumerate(_spread(case["n"], case["lo"], case["hi"]))]


def work(case):
    """Inputs read once, outputs written once; of the cache what the rows attend to."""
    k = case["kind"]
    if k == "plan":
        new = sum(max(0, a) for _, a in _steps(case))
        more = sum(_pages(l + a, case["page"]) - _pages(l, case["page"]) for l, a in _steps(case) if a > 0)
        freed = sum(_pages(l, case["page"]) for l, a in _steps(case) if a < 0)
        return {"bytes": 16 * case["n"] + 4 + 12 * (new + case["pad"]) + 8 * (more + freed), "flops": 0}
    D, H, KV = case["dim"], case["heads"], case["kv"]
    size = 2 if case["type"] == F16 else 4
    if k == "rope":
        T = case["rows"]
        return {"bytes": T * D * (4 * (H + 2 * KV) + 4 * H + size * 2 * KV) + 8 * T + (8 * D if case["norm"] else 0),
                "flops": T * (H + KV) * (4.0 * D + 3 * case["rot"])}
    lens, e = _lengths(case), case["each"]
    rows = case["n"] * e
    seen = sum(l * e - e * (e - 1) // 2 for l in lens if l)          # sum of the rows' lengths
    return {"bytes": sum(lens) * 2 * KV * D * size + rows * H * D * (12 if case["gate"] else 8), "flops": 4.0 * H * D * seen}


# ---- state -------------------------------------------------------------------
class _State:
    pass


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _perm(g, n):
    return torch.randperm(n, device="cuda", generator=g).to(torch.int32)


def _prepare_plan(s, case, g):
    n, page = case["n"], case["page"]
    steps = _steps(case)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(g.initial_seed())).tolist()
    steps = [steps[i] for i in order]
    used = [_pages(l, page) for l, _ in steps]
    s.width = max(_pages(l + max(0, a), page) for l, a in steps) + 3
    s.pool = int(1.3 * (sum(used) + sum(_pages(max(0, a), page) + 1 for _, a in steps))) + 5
    s.rows = sum(max(0, a) for _, a in steps) + case["pad"]
    s.page, s.n = page, n
    s.len, s.add = _ints([l for l, _ in steps]), _ints([a for _, a in steps])
    ids = _perm(g, s.pool)
    at = torch.cumsum(_ints([0] + used), 0).to(torch.int64)
    j = torch.arange(s.width, device="cuda")
    held = j < _ints(used)[:, None]
    s.table = torch.where(held, ids[(at[:-1, None] + j).clamp(max=s.pool - 1)], -1).to(torch.int32).contiguous()
    head, free = 7 * s.pool + 3, s.pool - sum(used)
    s.ring = torch.full((s.pool,), -1, dtype=torch.int32, device="cuda")
    s.ring[(head + torch.arange(free, device="cuda")) % s.pool] = ids[sum(used):]
    s.ctl = torch.tensor([head, head + free], dtype=torch.int64, device="cuda")


def _prepare_rope(s, case, g):
    T, H, KV, D = case["rows"] + case["pad"], case["heads"], case["kv"], case["dim"]
    s.valid, s.rot, s.adjacent, s.page = case["rows"], case["rot"], case["adjacent"], case["page"]
    # the query projection's rows hold each head's gate behind its query
    s.qg, s.k, s.v = 3 * _normal(g, T, H, 2, D), 2 * _normal(g, T, KV, D), _normal(g, T, KV, D)
    s.q_norm = s.k_norm = None
    if case["norm"]:
        s.q_norm, s.k_norm = 1 + 0.2 * _normal(g, D), 1 + 0.2 * _normal(g, D)
    s.pos = torch.randint(0, case["far"], (T,), dtype=torch.int32, device="cuda", generator=g)
    n_pages = _pages(2 * T, s.page)
    s.slot = _perm(g, n_pages * s.page)[:T].contiguous()
    if case["pad"]:
        s.pos[case["rows"]:] = -1
        s.slot[case["rows"]:] = -1
    s.q_out = torch.zeros(T, H, D, device="cuda")
    s.kc, s.vc = (_normal(g, n_pages, KV, s.page, D).to(DTYPE[case["type"]]) for _ in range(2))


def _prepare_attn(s, case, g):
    n, e, H, KV, D, page = (case[k] for k in ("n", "each", "heads", "kv", "dim", "page"))
    lens = _lengths(case)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(g.initial_seed())).tolist()
    lens = [lens[i] for i in order]
    s.n, s.each, s.page, s.valid, s.longest = n, e, page, n * e, max(lens)
    used = [_pages(l, page) for l in lens]
    s.width, pool = max(1, max(used)), sum(used) + 2
    ids = _perm(g, pool)
    at = torch.cumsum(_ints([0] + used), 0).to(torch.int64)
    j = torch.arange(s.width, device="cuda")
    s.table = torch.where(j < _ints(used)[:, None], ids[(at[:-1, None] + j).clamp(max=pool - 1)], -1).to(torch.int32).contiguous()
    T = n * e + case["pad"]
    s.row_req = _ints([r for r in range(n) for _ in range(e)] + [-1] * case["pad"])
    s.row_pos = _ints([l - e + i if l else -1 for l in lens for i in range(e)] + [-1] * case["pad"])
    # keys share a direction that queries look along by their own measure: flat and peaked rows
    way = _normal(g, KV, 1, D)
    s.kc = _normal(g, pool, KV, page, D)
    s.kc += 0.3 * _normal(g, pool, KV, page, 1) * way
    s.kc = s.kc.to(DTYPE[case["type"]])
    s.vc = _normal(g, pool, KV, page, D).to(DTYPE[case["type"]])
    s.q = _normal(g, T, H, D) + 0.5 * _normal(g, T, H, 1) * way.repeat_interleave(H // KV, 0).reshape(H, D)
    s.scale = D ** -0.5
    s.qg = _normal(g, T, H, 2, D) if case["gate"] else None
    s.out = torch.zeros(T, H, D, device="cuda")


def prepare(case, seed):
    s = _State()
    s.kind = case["kind"]
    g = _gen(seed)
    {"plan": _prepare_plan, "rope": _prepare_rope, "attn": _prepare_attn}[s.kind](s, case, g)
    if own:
        _bind(s, case)
    return s


def _bind(s, case):
    """The argument structures of the library's calls, and its output buffers."""
    import ctypes as C

    import roaster_amd as R
    L = R.lib()
    R.check(L.roaster_init(), "init")
    if s.kind == "plan":
        s.len_out, s.ctl_out = torch.empty_like(s.len), torch.empty_like(s.ctl)
        s.first = torch.empty(s.n + 1, dtype=torch.int32, device="cuda")
        s.row_req, s.row_pos, s.row_slot = (torch.empty(s.rows, dtype=torch.int32, device="cuda") for _ in range(3))
        a = R.RoasterKvPlan(s.n, s.page, s.pool, s.width, s.rows, R.ptr(s.len), R.ptr(s.add), R.ptr(s.len_out),
                            R.ptr(s.table), R.ptr(s.ring), R.ptr(s.ctl), R.ptr(s.ctl_out), R.ptr(s.first),
                            R.ptr(s.row_req), R.ptr(s.row_pos), R.ptr(s.row_slot))
        s.call, s.args = L.roaster_kv_plan, (C.byref(a),)
        s.keep = (a,)
        return
    c = R.RoasterKvCache(R.ptr(s.kc), R.ptr(s.vc), case["type"], s.kc.shape[0], case["page"], case["kv"], case["dim"])
    H, KV, D = case["heads"], case["kv"], case["dim"]
    if s.kind == "rope":
        a = R.RoasterQkRope(s.pos.numel(), H, R.ptr(s.qg), 2 * H * D, 2 * D, R.ptr(s.k), KV * D, D, R.ptr(s.v), KV * D, D,
                            R.ptr(s.q_norm), R.ptr(s.k_norm), EPS, s.rot, int(s.adjacent), THETA, R.ptr(s.pos),
                            R.ptr(s.slot), R.ptr(s.q_out))
        s.call = L.roaster_qk_rope_store
    else:
        s.ws = torch.empty(L.roaster_attn_ws_bytes(s.row_req.numel(), H, C.byref(c)), dtype=torch.uint8, device="cuda")
        gate = s.qg[:, :, 1] if case["gate"] else None
        a = R.RoasterAttnPaged(s.row_req.numel(), H, R.ptr(s.q), R.ptr(s.row_req), R.ptr(s.row_pos), R.ptr(s.table), s.n,
                               s.width, s.scale, R.ptr(gate), 2 * H * D, 2 * D, R.ptr(s.out), R.ptr(s.ws), s.ws.numel())
        s.call = L.roaster_attn_paged
    s.args = (C.byref(a), C.byref(c))
    s.keep = (a, c)


# ---- the operators, plainly ----------------------------------------------------
def _plan(s):
    dev, N = s.len.device, s.pool
    ln, add = s.len.long(), s.add.long()
    new, ended = add.clamp(min=0), add < 0
    have = (ln + s.page - 1) // s.page
    more = (ln + new + s.page - 1) // s.page - have
    gone = torch.where(ended, have, 0)
    zero = torch.zeros(1, dtype=torch.int64, device=dev)
    first, pages, freed = (torch.cat([zero, torch.cumsum(v, 0)]) for v in (new, more, gone))
    head, tail = s.ctl[0], s.ctl[1]
    j = torch.arange(s.width, device=dev)[None, :]
    at = j - have[:, None]
    taken = s.ring[(head + pages[:-1, None] + at) % N]
    table = torch.where((at >= 0) & (at < more[:, None]), taken, s.table)
    back = torch.where(j < gone[:, None], (tail + freed[:-1, None] + j) % N, N)     # entry N takes what is not given back
    ring = torch.cat([s.ring, s.ring[:1]]).scatter(0, back.reshape(-1), s.table.reshape(-1))[:N]
    t = torch.arange(s.rows, device=dev)
    r = torch.searchsorted(first[1:], t, right=True)
    real = r < s.n
    r = r.clamp(max=s.n - 1)
    pos = ln[r] + t - first[r]
    slot = table[r, (pos // s.page).clamp(max=s.width - 1)] * s.page + pos % s.page
    rows = [torch.where(real, v, -1).to(torch.int32) for v in (r, pos, slot)]
    ctl = torch.stack([head + pages[-1], tail + freed[-1]])
    return [table, ring, torch.where(ended, 0, ln + new).to(torch.int32), ctl, first.to(torch.int32)] + rows


def _rotate(x, cos, sin, adjacent):
    """x [T, heads, rot] rotated by pairs: (i, i + rot/2), or (2i, 2i + 1)."""
    a, b = (x[..., 0::2], x[..., 1::2]) if adjacent else x.chunk(2, dim=-1)
    y = (a * cos - b * sin, b * cos + a * sin)
    return torch.stack(y, dim=-1).flatten(-2) if adjacent else torch.cat(y, dim=-1)


def _normed(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * w


def _rope(s):
    T, rot = s.valid, s.rot
    i = torch.arange(rot // 2, device=s.pos.device, dtype=torch.float64)
    angle = s.pos[:T, None, None].double() * THETA ** (-2 * i / rot)
    cos, sin = angle.cos().float(), angle.sin().float()
    out = [_normed(s.qg[:T, :, 0], s.q_norm), _normed(s.k[:T], s.k_norm)]
    out = [torch.cat([_rotate(x[..., :rot], cos, sin, s.adjacent), x[..., rot:]], dim=-1) for x in out]
    s.q_out[:T] = out[0]
    at = s.slot[:T].long()
    s.kc[at // s.page, :, at % s.page] = out[1].to(s.kc.dtype)
    s.vc[at // s.page, :, at % s.page] = s.v[:T].to(s.vc.dtype)
    return [s.q_out, s.kc, s.vc]


def _attn(s):
    n, e, L = s.n, s.each, s.longest
    H, D = s.q.shape[1:]
    KV = s.kc.shape[1]
    j = torch.arange(L, device=s.q.device)
    page = s.table[:, j // s.page].clamp(min=0).long()
    k, v = (c[page, :, j % s.page].float().transpose(1, 2).contiguous() for c in (s.kc, s.vc))   # [n, KV, L, D]
    q = s.q[:n * e].reshape(n, e, KV, H // KV, D).permute(0, 2, 1, 3, 4).reshape(n, KV, e * (H // KV), D)
    score = (q @ k.transpose(-1, -2).contiguous()) * s.scale
    pos = s.row_pos[:n * e].reshape(n, 1, e, 1).expand(n, 1, e, H // KV).reshape(n, 1, -1, 1)
    seen = j <= pos
    score = score.masked_fill(~seen, -math.inf)
    p = torch.exp(score - score.amax(dim=-1, keepdim=True).clamp(min=-1e30)).masked_fill(~seen, 0)
    v = v.masked_fill(~seen.any(dim=-2).unsqueeze(-1), 0)
    o = (p @ v) / p.sum(dim=-1, keepdim=True).clamp(min=1e-30)
    o = o.reshape(n, KV, e, H // KV, D).permute(0, 2, 1, 3, 4).reshape(n * e, H, D)
    if s.qg is not None:
        o = o / (1 + torch.exp(-s.qg[:n * e, :, 1]))
    s.out[:n * e] = o
    return s.out


def run(s):
    if own:
        rc = s.call(*s.args)
        if rc:
            raise RuntimeError("call failed (%d)" % rc)
        if s.kind == "plan":
            return [s.table, s.ring, s.len_out, s.ctl_out, s.first, s.row_req, s.row_pos, s.row_slot]
        return [s.q_out, s.kc, s.vc] if s.kind == "rope" else s.out
    return {"plan": _plan, "rope": _rope, "attn": _attn}[s.kind](s)


# ---- the same in 64 bits -----------------------------------------------------
def _exact_plan(s):
    """Request by request, on the host."""
    table, ring = s.table.cpu().numpy().copy(), s.ring.cpu().numpy().copy()
    head, tail = s.ctl.tolist()
    rows, first, after = [], [0], []
    for r, (l, a) in enumerate(zip(s.len.tolist(), s.add.tolist())):
        have = -(-l // s.page)
        if a < 0:
            for p in table[r, :have]:
                ring[tail % s.pool] = p
                tail += 1
        for p in range(l, l + max(0, a)):
            if p // s.page >= have:
                table[r, have] = ring[head % s.pool]
                head, have = head + 1, have + 1
            rows.append((r, p, int(table[r, p // s.page]) * s.page + p % s.page))
        first.append(len(rows))
        after.append(0 if a < 0 else l + a)
    rows += [(-1, -1, -1)] * (s.rows - len(rows))
    cols = [_ints([v[i] for v in rows]) for i in range(3)]
    ctl = torch.tensor([head, tail], dtype=torch.int64, device="cuda")
    return [torch.from_numpy(table).cuda(), torch.from_numpy(ring).cuda(), _ints(after), ctl, _ints(first)] + cols


def _exact_rope(s):
    """As products of complex numbers."""
    T, half = s.valid, s.rot // 2
    inv = torch.exp(-math.log(THETA) * torch.arange(half, device="cuda", dtype=torch.float64) / half)
    turn = torch.polar(torch.ones(T, 1, half, device="cuda", dtype=torch.float64), s.pos[:T].double().view(T, 1, 1) * inv)
    q, k, v = s.q_out.double(), s.kc.double(), s.vc.double()
    got = []
    for x, w in ((s.qg[:T, :, 0].double(), s.q_norm), (s.k[:T].double(), s.k_norm)):
        if w is not None:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()
        x = x.clone()
        lo, hi = (slice(0, s.rot, 2), slice(1, s.rot, 2)) if s.adjacent else (slice(0, half), slice(half, s.rot))
        z = torch.complex(x[..., lo], x[..., hi]) * turn
        x[..., lo], x[..., hi] = z.real, z.imag
        got.append(x)
    q[:T] = got[0]
    flat = lambda c: c.transpose(1, 2).reshape(-1, c.shape[1], c.shape[3])  # noqa: E731  [slot, KV, D]
    for c, new in ((k, got[1]), (v, s.v[:T].double())):
        f = flat(c).clone()
        f[s.slot[:T].long()] = new
        c.copy_(f.view(c.shape[0], s.page, c.shape[1], c.shape[3]).transpose(1, 2))
    return [q, k, v]


def _exact_attn(s):
    """Row by row over the row's own tokens (rows of one request together)."""
    H, D = s.q.shape[1:]
    KV, e = s.kc.shape[1], s.each
    out = s.out.double()
    for r in range(s.n):
        rows = slice(r * e, (r + 1) * e)
        pos = s.row_pos[rows].tolist()
        last = max(pos) + 1
        if not last:
            continue
        pages = s.table[r, :_pages(last, s.page)].long()
        k, v = (c[pages].transpose(0, 1).reshape(KV, -1, D)[:, :last].double() for c in (s.kc, s.vc))
        q = s.q[rows].double().reshape(e, KV, H // KV, D)
        for h in range(KV):
            score = (q[:, h].reshape(-1, D) @ k[h].T * s.scale).reshape(e, H // KV, last)
            late = torch.arange(last, device="cuda")[None, :] > s.row_pos[rows, None]
            p = torch.softmax(score.masked_fill(late[:, None, :], -math.inf), dim=-1)
            out[rows].view(e, KV, H // KV, D)[:, h] = (p.reshape(-1, last) @ v[h]).reshape(e, H // KV, D)
    if s.qg is not None:
        T = s.n * e
        out[:T] *= torch.sigmoid(s.qg[:T, :, 1].double())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "rope": _exact_rope, "attn": _exact_attn}[s.kind](s)
