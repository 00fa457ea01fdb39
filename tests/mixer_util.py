"""Plain 64-bit forms of the operators of a recurrent layer (include/roaster_mixer.h),
the bounds that their tests hold results to, and the device state they share."""
import ctypes as C

import numpy as np

import roaster_amd as R
from attn_util import EPS24, sync  # noqa: F401
from gpu_util import Dev


def sigmoid(x):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-x))


# ---- norm --------------------------------------------------------------------
def norm_oracle(v, group, weight, gate, eps):
    """y of rows v (x, or the residual after the addition)."""
    v = v.astype(np.float64)
    y = v
    if group:
        h = v.reshape(v.shape[0], -1, group)
        y = h / np.sqrt((h * h).mean(axis=2, keepdims=True) + eps)
        y = (y if weight is None else y * weight.astype(np.float64)).reshape(v.shape)
    if gate is not None:
        g = gate.astype(np.float64)
        y = y * (g * sigmoid(g))
    return y


def eights(y):
    """The values and scales in 8 bits of f32 rows, as the header has them, every step in f32."""
    top = np.abs(y).max(axis=1)
    live = top >= 2.0 ** -119
    mul = np.float32(127) / np.where(live, top, 1).astype(np.float32)
    q = np.where(live[:, None], np.rint(y * mul[:, None]), 0).astype(np.int8)
    return q, np.where(live, top / np.float32(127), 0).astype(np.float32)


# ---- product -----------------------------------------------------------------
def unpacked(data, rows, cols):
    """int8 [rows][cols] out of the order of the products, and that its padding is zero."""
    rp, cp = -(-rows // 32) * 32, -(-cols // 128) * 128
    v = data.view(np.int8).reshape(rp // 32, cp // 16, 32, 16).transpose(0, 2, 1, 3).reshape(rp, cp)
    assert not v[rows:].any() and not v[:, cols:].any()
    return v[:rows, :cols]


def packed(wq):
    """The order of the products, on the host."""
    rows, cols = wq.shape
    v = np.zeros((-(-rows // 32) * 32, -(-cols // 128) * 128), np.int8)
    v[:rows, :cols] = wq
    return np.ascontiguousarray(v.reshape(v.shape[0] // 32, 32, v.shape[1] // 16, 16).transpose(0, 2, 1, 3))


# ---- scan --------------------------------------------------------------------
class Scan:
    """A scan's inputs on the host: sizes, weights, states and rows."""

    def __init__(self, rng, new, pos, mode=R.SCAN_DELTA, kh=2, vh=4, kd=64, vd=64, taps=4, pad=0, bias=True, dt_bias=True, skip=True,
                 wide=0, scale=None):
        self.new, self.pos, self.mode, self.kh, self.vh, self.kd, self.vd, self.taps = list(new), list(pos), mode, kh, vh, kd, vd, taps
        self.n, self.C = len(new), 2 * kh * kd + vh * vd
        T = sum(new)
        self.T, self.rows = T, max(1, T + pad)
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.x, self.a, self.b = f(self.rows, self.C + 4 * wide), f(self.rows, vh + wide), f(self.rows, vh + 2 * wide)
        self.conv_w, self.conv_b = f(self.C, taps) / np.float32(np.sqrt(taps)), 0.1 * f(self.C) if bias else None
        self.a_coef = -np.exp(rng.uniform(0, np.log(16), vh)).astype(np.float32)
        self.dt_bias = rng.uniform(-6, -1, vh).astype(np.float32) if dt_bias else None
        self.skip = f(vh) if skip else None
        self.conv, self.state = f(self.n, taps, self.C), 0.3 * f(self.n, vh, vd, kd)
        self.scale = scale if scale is not None else (kd ** -0.5 if mode == R.SCAN_DELTA else 0.7)
        self.eps = 1e-6
        self.first = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.row_pos = np.array([p + i for m, p in zip(new, pos) for i in range(m)] + [-1] * (self.rows - T), np.int32)
        self.wide = wide

    def most(self):
        return max([1] + self.new)


def scan_oracle(s):
    """Token by token in 64 bits: out, conv, state, and bounds of the f32 results' errors of out and state.

    The bounds follow a value element's row of the state (its norm, and the mass m of what has been added to it,
    decayed) through the recurrence, in which the correction only shrinks errors.  A channel of the convolution is
    off by taps + 2 roundings of the sum of its terms' sizes (silu's slope is at most 1.1) and 6 of itself; a unit vector by its
    channels' errors and KD + 8 roundings; a step's other roundings are those of sums of up to KD and 64 terms (a prompt's
    tokens are taken 64 at a time), twice since each of them enters the solution and the product with it."""
    e = EPS24
    rep, nk = s.vh // s.kh, s.kh * s.kd
    loc = 2 * (s.kd + 64 + 16) * e
    out = np.full((s.rows, s.vh, s.vd), 77.0)
    oerr = np.zeros(out.shape)
    conv, state, serr = s.conv.astype(np.float64), s.state.astype(np.float64), np.zeros((s.n, s.vh, s.vd))
    w = s.conv_w.astype(np.float64)
    for r in range(s.n):
        if not s.new[r]:
            continue
        f0, p0 = s.first[r], s.pos[r]
        S = state[r] if p0 else np.zeros_like(state[r])
        E = np.zeros((s.vh, s.vd))
        m = np.linalg.norm(S, axis=2)
        hist = [conv[r, (p0 - i) % s.taps].copy() if p0 >= i else np.zeros(s.C) for i in range(s.taps - 1, 0, -1)]
        for i in range(s.new[r]):
            x = s.x[f0 + i, :s.C].astype(np.float64)
            win = np.stack(hist + [x])                     # [taps, C]
            c = (w.T * win).sum(axis=0) + (0 if s.conv_b is None else s.conv_b)
            size = (np.abs(w.T) * np.abs(win)).sum(axis=0) + (0 if s.conv_b is None else np.abs(s.conv_b))
            c = c * sigmoid(c)
            ce = e * (1.1 * (s.taps + 2) * size + 6 * np.abs(c))
            q, k = (np.repeat(c[j * nk:(j + 1) * nk].reshape(s.kh, s.kd), rep, axis=0) for j in (0, 1))
            qe, ke = (np.repeat(np.linalg.norm(ce[j * nk:(j + 1) * nk].reshape(s.kh, s.kd), axis=1), rep) for j in (0, 1))
            v, ve = c[2 * nk:].reshape(s.vh, s.vd), ce[2 * nk:].reshape(s.vh, s.vd)
            a = s.a[f0 + i, :s.vh].astype(np.float64) + (0 if s.dt_bias is None else s.dt_bias)
            dt = np.maximum(a, 0) + np.log1p(np.exp(-np.abs(a)))
            g = s.a_coef.astype(np.float64) * dt
            d, de = np.exp(g)[:, None], (e * (4 + 8 * np.abs(g)))[:, None]
            # dt = log(1 + e^a): a's own rounding is as large in it as in a
            dte = e * (6 + np.abs(a) / np.maximum(dt, 1e-30) * np.minimum(1, np.exp(a)))
            if s.mode == R.SCAN_DELTA:
                qn, kn = (np.sqrt((z * z).sum(axis=1) + s.eps) for z in (q, k))
                q, k = q / qn[:, None], k / kn[:, None]
                qe, ke = qe / qn + (s.kd + 8) * e, ke / kn + (s.kd + 8) * e
                gain = sigmoid(s.b[f0 + i, :s.vh].astype(np.float64))[:, None]
                wv = gain * (v - d * np.einsum("hvk,hk->hv", S, k))
                we = gain * (ve + d * m * ke[:, None] + d * m * de) + np.abs(wv) * 8 * e
                kn = np.ones(s.vh)
            else:
                gain = dt[:, None]
                wv = gain * v
                we = gain * ve + np.abs(wv) * dte[:, None]
                kn = np.linalg.norm(k, axis=1)
                qe, ke = qe + 2 * e * np.linalg.norm(q, axis=1), ke + 2 * e * kn
            de = de + np.abs(g)[:, None] * dte[:, None]
            S = d[..., None] * S + wv[..., None] * k[:, None, :]
            add = np.abs(wv) * kn[:, None]
            m = d * m + add
            E = d * E + d * m * de + we * kn[:, None] + np.abs(wv) * ke[:, None] + loc * m
            o = s.scale * np.einsum("hvk,hk->hv", S, q)
            qn = np.linalg.norm(q, axis=1)[:, None]
            oe = abs(s.scale) * (qn * (E + loc * m) + m * qe[:, None])
            if s.skip is not None:
                o = o + s.skip.astype(np.float64)[:, None] * v
                oe = oe + np.abs(s.skip)[:, None] * ve + 2 * e * np.abs(o) + 2 * e * np.abs(s.skip[:, None] * v)
            out[f0 + i], oerr[f0 + i] = o, oe
            hist = hist[1:] + [x]
        for i in range(max(0, s.new[r] - s.taps), s.new[r]):
            conv[r, (p0 + i) % s.taps] = s.x[f0 + i, :s.C]
        state[r], serr[r] = S, E + 2 * e * m
    return out, conv, state, oerr, serr


class ScanCall:
    """A scan's device state and its call."""

    def __init__(self, s, most=None, ws_extra=0, **kw):
        self.s = s
        self.d = {k: Dev(getattr(s, k)) for k in ("x", "a", "b", "conv_w", "a_coef", "first", "row_pos", "conv", "state")}
        for k in ("conv_b", "dt_bias", "skip"):
            self.d[k] = Dev(getattr(s, k)) if getattr(s, k) is not None else None
        self.out = Dev(np.full((s.rows, s.vh, s.vd), 77, np.float32))
        p = lambda k: self.d[k].p if self.d[k] else None  # noqa: E731
        self.st = R.RoasterSsmState(s.n, s.kh, s.vh, s.kd, s.vd, s.taps, p("conv"), p("state"))
        most = s.most() if most is None else most
        need = R.lib().roaster_ssm_ws_bytes(s.rows, most, C.byref(self.st))
        assert need
        self.ws = Dev(np.full(need + ws_extra, 0xFF, np.uint8))           # NaN where it is read as f32
        a = dict(rows=s.rows, most=most, mode=s.mode, x=p("x"), x_row=s.x.shape[1], a=p("a"), a_row=s.a.shape[1], b=p("b"),
                 b_row=s.b.shape[1], conv_w=p("conv_w"), conv_b=p("conv_b"), a_coef=p("a_coef"), dt_bias=p("dt_bias"), skip=p("skip"),
                 scale=s.scale, eps=s.eps, first=p("first"), row_pos=p("row_pos"), out=self.out.p, out_row=s.vh * s.vd, ws=self.ws.p,
                 ws_bytes=need)
        a.update(kw)
        self.a = R.RoasterSsmScan(**a)

    def call(self):
        return R.lib().roaster_ssm_scan(C.byref(self.a), C.byref(self.st))

    def got(self):
        return self.out.get(), self.d["conv"].get(), self.d["state"].get()


def check_scan(got, want):
    """The largest share of their bounds that out and state use; conv exactly."""
    out, conv, state = got
    o, c, s, oe, se = want
    assert np.array_equal(conv.astype(np.float64), c)
    err, lim = np.abs(out - o), oe + 1e-30
    assert np.all(err <= lim), ("out", float(np.nanmax(err / lim)), np.argwhere(~(err <= lim))[:4].tolist())
    es, ls = np.linalg.norm(state - s, axis=3), se + 1e-30
    assert np.all(es <= ls), ("state", float(np.nanmax(es / ls)), np.argwhere(~(es <= ls))[:4].tolist())
    return float((err / lim).max()), float((es / ls).max())
