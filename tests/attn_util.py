"""Plain 64-bit forms of the attention operators (include/roaster_attn.h) and the
device state their tests share."""
import ctypes as C

import numpy as np

import roaster_amd as R
from gpu_util import Dev

EPS24 = 2.0 ** -24                  # half a step of f32, relative


def sync():
    R.check(R.lib().roaster_sync(), "sync")


# ---- plan --------------------------------------------------------------------
def plan_oracle(page, n_pages, max_rows, ln, add, table, ring, ctl):
    """Request by request; the state after the step and its rows."""
    table, ring = table.copy(), ring.copy()
    front, end = int(ctl[0]), int(ctl[1])
    rows, first, after = [], [0], []
    for r, (l, a) in enumerate(zip(ln.tolist(), add.tolist())):
        have = -(-l // page)
        if a < 0:
            for p in table[r, :have]:
                ring[end % n_pages] = p
                end += 1
        for pos in range(l, l + max(a, 0)):
            if pos // page >= have:
                table[r, have] = ring[front % n_pages]
                front, have = front + 1, have + 1
            rows.append((r, pos, int(table[r, pos // page]) * page + pos % page))
        first.append(len(rows))
        after.append(0 if a < 0 else l + a)
    rows += [(-1, -1, -1)] * (max_rows - len(rows))
    rows = np.array(rows, np.int32)
    return dict(len_out=np.array(after, np.int32), table=table, ring=ring, ctl_out=np.array([front, end], np.int64),
                first=np.array(first, np.int32), row_req=rows[:, 0], row_pos=rows[:, 1], row_slot=rows[:, 2])


class Plan:
    """A plan's device state and its call."""

    def __init__(self, page, n_pages, max_rows, ln, add, table, ring, ctl, in_place=False):
        ln, add = np.asarray(ln, np.int32), np.asarray(add, np.int32)
        n = len(ln)
        self.len, self.add, self.table, self.ring, self.ctl = (Dev(a) for a in (ln, add, table, ring, ctl))
        self.len_out = self.len if in_place else Dev(np.full(n, 77, np.int32))
        self.ctl_out = self.ctl if in_place else Dev(np.full(2, 77, np.int64))
        self.first = Dev(np.full(n + 1, 77, np.int32))
        self.row_req, self.row_pos, self.row_slot = (Dev(np.full(max_rows, 77, np.int32)) for _ in range(3))
        self.a = R.RoasterKvPlan(n, page, n_pages, table.shape[1], max_rows, self.len.p, self.add.p, self.len_out.p,
                                 self.table.p, self.ring.p, self.ctl.p, self.ctl_out.p, self.first.p, self.row_req.p,
                                 self.row_pos.p, self.row_slot.p)

    def call(self):
        return R.lib().roaster_kv_plan(C.byref(self.a))

    def got(self):
        return {k: getattr(self, k).get() for k in ("len_out", "table", "ring", "ctl_out", "first", "row_req",
                                                   "row_pos", "row_slot")}


def pool(rng, page, ln, more, width, slack=3, front=0):
    """Tables of the requests' pages out of a shuffled pool, the rest of it in the ring."""
    used = [-(-int(l) // page) for l in ln]
    n_pages = sum(used) + more + slack
    ids = rng.permutation(n_pages).astype(np.int32)
    table = np.full((len(ln), width), -1, np.int32)
    at = 0
    for r, u in enumerate(used):
        table[r, :u] = ids[at:at + u]
        at += u
    free = n_pages - at
    ring = np.full(n_pages, -1, np.int32)
    ring[(front + np.arange(free)) % n_pages] = ids[at:]
    return n_pages, table, ring, np.array([front, front + free], np.int64)


# ---- norms and rotation ----------------------------------------------------------
def rope_oracle(x, w, pos, eps, rot, adjacent, theta):
    """x [T, heads, D] in 64 bits, and the size of each element's pair (what its rounding goes by)."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * w.astype(np.float64)
    size = np.abs(x)
    y, size = x.copy(), size.copy()
    h = rot // 2
    if h:
        lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if adjacent else (slice(0, h), slice(h, rot))
        ang = pos[:, None, None].astype(np.float64) * np.float64(theta) ** (-2.0 * np.arange(h) / rot)
        a, b = x[..., lo], x[..., hi]
        y[..., lo], y[..., hi] = a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang)
        size[..., lo] = size[..., hi] = np.abs(a) + np.abs(b)
    return y, size


# ---- attention -----------------------------------------------------------------
def attn_oracle(q, kc, vc, table, row_req, row_pos, scale, gate=None):
    """Outputs in 64 bits, sum_j p_j |v_j| and max_j scale |q| . |k_j| per row and head (what
    rounding errors go by).  kc, vc: [n_pages, kv, page, D]."""
    T, H, D = q.shape
    KV, page = kc.shape[1], kc.shape[2]
    out, mass, reach = np.zeros((T, H, D)), np.zeros((T, H, D)), np.zeros((T, H))
    q = q.astype(np.float64)
    for t in range(T):
        n = int(row_pos[t]) + 1
        if row_req[t] < 0 or n <= 0:
            continue
        pages = table[row_req[t], :-(-n // page)]
        k, v = (c[pages].transpose(1, 0, 2, 3).reshape(KV, -1, D)[:, :n].astype(np.float64) for c in (kc, vc))
        for h in range(H):
            g = h // (H // KV)
            s = k[g] @ q[t, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[t, h], mass[t, h] = p @ v[g], p @ np.abs(v[g])
            reach[t, h] = (np.abs(k[g]) @ np.abs(q[t, h])).max() * abs(scale)
    if gate is not None:
        s = 1 / (1 + np.exp(-gate.astype(np.float64)))
        out, mass = out * s, mass * s
    return out, mass, reach


class Cache:
    """A layer's cache on the device from host arrays [n_pages, kv, page, D]."""

    def __init__(self, kc, vc):
        self.k, self.v = Dev(kc), Dev(vc)
        self.c = R.RoasterKvCache(self.k.p, self.v.p, R.KV_F16 if kc.dtype == np.float16 else R.KV_F32, kc.shape[0],
                                  kc.shape[2], kc.shape[1], kc.shape[3])


class Attn:
    """An attention call: its device buffers, the outputs first filled with 77."""

    def __init__(self, cache, q, row_req, row_pos, table, scale, gate=None, rows=None):
        T, H, D = q.shape
        self.cache = cache
        self.q, self.req, self.pos, self.table = (Dev(a) for a in (q, row_req, row_pos, table))
        self.gate = Dev(gate) if gate is not None else None       # [T, H, 2, D]: the second of each pair
        self.out = Dev(np.full((T, H, D), 77, np.float32))
        need = R.lib().roaster_attn_ws_bytes(T, H, C.byref(cache.c))
        assert need > 0
        self.ws = Dev(np.full(need // 4 + 1, np.nan, np.float32))
        self.a = R.RoasterAttnPaged(T if rows is None else rows, H, self.q.p, self.req.p, self.pos.p, self.table.p,
                                    table.shape[0], table.shape[1], scale,
                                    self.gate.p + 4 * D if gate is not None else None, 2 * H * D, 2 * D, self.out.p,
                                    self.ws.p, need)

    def call(self):
        return R.lib().roaster_attn_paged(C.byref(self.a), C.byref(self.cache.c))


def attn_bound(mass, reach, n, D):
    """How far an output element may be from the 64-bit one.  A score is a sum of D
    products, its terms off by at most 2^-22 (a query in two fp16 parts, or its
    product with scale and log2 e in f32) and its sum by D + 2 roundings; the
    softmax weights are off by twice the score's error, 2^-22 each for being
    split, 8 roundings for exp and the division; the sum over n positions by n + 8
    roundings, each of at most 2^-24 of sum p |v|."""
    ds = reach * (2.0 ** -22 + (D + 2) * EPS24)
    return mass * (2 * ds[..., None] + 2.0 ** -21 + (n + 16) * EPS24) + 1e-30


def check_attn(got, want, mass, reach, n, D):
    err = np.abs(got - want)
    lim = attn_bound(mass, reach, n, D)
    assert np.all(err <= lim), (float((err / lim).max()), np.unravel_index(np.argmax(err / lim), err.shape))
    # as a whole: an operand rounded once to fp16 would show as 1e-4 or more
    norm = np.linalg.norm(want)
    rel = np.linalg.norm(got - want) / norm if norm else np.linalg.norm(got - want)
    assert rel <= 1e-5, rel
    return rel
