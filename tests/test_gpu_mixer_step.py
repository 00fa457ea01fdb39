"""The operators of a recurrent layer as a serving step uses them together: plan, norm with the
residual, projections in 8 bits, scan, norm over heads with its gate, output projection, norm, the MoE block
-- each step against 64-bit arithmetic on the host, and the steps of a captured graph against the same
calls made eagerly."""
import ctypes as C

import numpy as np
import pytest

import roaster_amd as R
from attn_util import EPS24, Attn, Cache, Plan, plan_oracle, pool, sync
from gpu_util import Dev, SynthTable, log
from mixer_util import Scan, ScanCall, check_scan, norm_oracle, scan_oracle, unpacked
from test_gpu_attn_step import Graph
from test_gpu_norm import REL

pytestmark = pytest.mark.gpu
HID, KH, VH, KD, VD, TAPS, EPS = 2048, 2, 4, 128, 128, 4, 1e-6
CH, VALUES = 2 * KH * KD + VH * VD, VH * VD
WIDE = CH + VALUES                                           # the scan's channels, then the gate


def pack(W, frm, rows, cols):
    """The matrix on the device, and its values and scales on the host."""
    d = [Dev(W), Dev(nbytes=R.lib().roaster_i8_bytes(rows, cols), dtype=np.int8), Dev(nbytes=4 * rows)]
    w = R.RoasterI8(d[1].p, d[2].p, rows, cols)
    R.check(R.lib().roaster_i8_pack(d[0].p, frm, C.byref(w)), "pack")
    sync()
    return w, d


class Layer:
    """One layer's weights, and a step's calls on buffers of `rows` rows."""

    def __init__(self, rng):
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        n = WIDE * (HID // 256)
        self.q4, self.q6 = R.synth_q4k(5, 1, n, 5e-5, 2e-4), R.synth_q6k(5, 2, HID * (VALUES // 256), 3e-5, 9e-5)
        self.small = f(2 * VH, HID) / np.float32(np.sqrt(HID))
        self.w_in, self.w_ab, self.w_out = (pack(self.q4, R.I8_FROM_Q4K, WIDE, HID), pack(self.small, R.I8_FROM_F32, 2 * VH, HID),
                                            pack(self.q6, R.I8_FROM_Q6K, HID, VALUES))
        self.norms = [1 + 0.2 * f(HID), 1 + 0.2 * f(VD), 1 + 0.2 * f(HID)]
        self.d_norms = [Dev(v) for v in self.norms]


class Step:
    def __init__(self, layer, s, rows, most, plan):
        """s: a Scan that gives the states and the scan's weights."""
        L, self.layer, self.s, self.rows, self.plan = R.lib(), layer, s, rows, plan
        f = lambda *sh: Dev(np.full(sh, 77, np.float32))  # noqa: E731
        self.x, self.h = f(rows, HID), f(rows, HID)
        eight = lambda *sh: Dev(np.full(sh, 77, np.int8))  # noqa: E731
        self.q1, self.s1, self.wide, self.ab, self.mix = eight(rows, HID), f(rows), f(rows, WIDE), f(rows, 2 * VH), f(rows, VH, VD)
        self.q2, self.s2, self.o, self.y = eight(rows, VALUES), f(rows), f(rows, HID), f(rows, HID)
        self.w = {k: Dev(getattr(s, k)) for k in ("conv_w", "conv_b", "a_coef", "dt_bias", "skip", "conv", "state")}
        self.st = R.RoasterSsmState(s.n, KH, VH, KD, VD, TAPS, self.w["conv"].p, self.w["state"].p)
        need = L.roaster_ssm_ws_bytes(rows, most, C.byref(self.st))
        self.ws = Dev(np.full(need, 0xFF, np.uint8))
        n1, n2, n3 = (d.p for d in layer.d_norms)
        p = lambda k: self.w[k].p  # noqa: E731
        self.a = [
            R.RoasterNorm(rows, HID, HID, self.x.p, HID, self.h.p, HID, n1, None, 0, EPS, None, 0, self.q1.p, HID, self.s1.p),
            R.RoasterMatmulI8(rows, self.q1.p, HID, self.s1.p, self.wide.p, WIDE),
            R.RoasterMatmulI8(rows, self.q1.p, HID, self.s1.p, self.ab.p, 2 * VH),
            R.RoasterSsmScan(rows, most, R.SCAN_DELTA, self.wide.p, WIDE, self.ab.p, 2 * VH, self.ab.p + 4 * VH, 2 * VH, p("conv_w"), p("conv_b"),
                             p("a_coef"), p("dt_bias"), p("skip"), s.scale, s.eps, plan.first.p, plan.row_pos.p, self.mix.p, VALUES, self.ws.p, need),
            R.RoasterNorm(rows, VALUES, VD, self.mix.p, VALUES, None, 0, n2, self.wide.p + 4 * CH, WIDE, EPS, None, 0, self.q2.p, VALUES, self.s2.p),
            R.RoasterMatmulI8(rows, self.q2.p, VALUES, self.s2.p, self.o.p, HID),
            R.RoasterNorm(rows, HID, HID, self.o.p, HID, self.h.p, HID, n3, None, 0, EPS, self.y.p, HID, None, 0, None)]

    def calls(self):
        L, a, w, r = R.lib(), self.a, self.layer, C.byref
        return [self.plan.call, lambda: L.roaster_norm(r(a[0])), lambda: L.roaster_matmul_i8(r(a[1]), r(w.w_in[0])),
                lambda: L.roaster_matmul_i8(r(a[2]), r(w.w_ab[0])), lambda: L.roaster_ssm_scan(r(a[3]), r(self.st)),
                lambda: L.roaster_norm(r(a[4])), lambda: L.roaster_matmul_i8(r(a[5]), r(w.w_out[0])), lambda: L.roaster_norm(r(a[6]))]

    def feed(self, x, h, add):
        for d, v in ((self.x, x), (self.h, h), (self.plan.add, np.asarray(add, np.int32))):
            R.check(R.lib().roaster_h2d(d.p, v.ctypes.data, v.nbytes), "h2d")

    def got(self):
        out = {k: getattr(self, k).get() for k in ("h", "q1", "s1", "wide", "ab", "mix", "q2", "s2", "o", "y")}
        return dict(out, conv=self.w["conv"].get(), state=self.w["state"].get(), **self.plan.got())


def product(q, scale, w):
    """The exact product of 8-bit rows with a packed matrix, and the bound of the f32 result's error."""
    d = w[1]
    v = unpacked(d[1].get(), w[0].rows, w[0].cols).astype(np.float64)
    y = (q.astype(np.float64) @ v.T) * scale[:, None].astype(np.float64) * d[2].get().astype(np.float64)
    return y, 3 * EPS24 * 1.01 * np.abs(y)


def check_eights(q, scale, y):
    """Values and scales against 64-bit rows: half a step and what the row's bound moves."""
    top = np.abs(y).max(axis=1)
    assert np.all(np.abs(scale - top / 127) <= (REL + 2 * EPS24) * top / 127)
    assert np.all(np.abs(q - y * (127 / top)[:, None]) <= 0.5 + 127 * (2 * REL + 4 * EPS24))


@pytest.fixture(scope="module")
def layer():
    return Layer(np.random.default_rng(41))


def check_step(layer, g, x, h, T, s, new, pos, conv, state):
    """Each stage from what the device gave the one before."""
    v = (x + h)[:T]
    n1, n2, n3 = layer.norms
    check_eights(g["q1"][:T], g["s1"][:T], norm_oracle(v, HID, n1, None, EPS))
    for name, w in (("wide", layer.w_in), ("ab", layer.w_ab)):
        y, lim = product(g["q1"][:T], g["s1"][:T], w)
        assert np.all(np.abs(g[name][:T] - y) <= lim), name
    s.new, s.pos, s.conv, s.state = list(new), list(pos), conv, state
    s.T = s.rows = T
    s.x, s.a, s.b = g["wide"][:T], g["ab"][:T, :VH], g["ab"][:T, VH:]
    s.first = g["first"]
    share = check_scan((g["mix"][:T], g["conv"], g["state"]), scan_oracle(s))
    gate = np.ascontiguousarray(g["wide"][:T, CH:])
    check_eights(g["q2"][:T], g["s2"][:T], norm_oracle(g["mix"][:T].reshape(T, VALUES), VD, n2, gate, EPS))
    o, lim = product(g["q2"][:T], g["s2"][:T], layer.w_out)
    assert np.all(np.abs(g["o"][:T] - o) <= lim)
    after = v + g["o"][:T]
    assert np.array_equal(g["h"][:T], after)
    want = norm_oracle(after, HID, n3, None, EPS)
    assert np.all(np.abs(g["y"][:T] - want) <= REL * np.abs(want) + 1e-37)
    return share


def test_serving_steps_of_one_layer(layer):
    """Three requests: prompts of 5, 90 and 17 tokens, a step of one token each, a step in which the first ends, the
    second adds one and the third seven, and one in which another request begins in the first's place."""
    rng = np.random.default_rng(42)
    rows, n = 120, 3
    s = Scan(rng, [1] * n, [0] * n, R.SCAN_DELTA, KH, VH, KD, VD, TAPS)
    page, width = 16, 16
    n_pages, table, ring, ctl = pool(rng, page, np.zeros(n, np.int32), 20, width, slack=0)
    ln, table_moe = np.zeros(n, np.int32), SynthTable(3, n_layers=1)
    conv, state = s.conv.copy(), s.state.copy()
    try:
        for add in ([5, 90, 17], [1, 1, 1], [-1, 1, 7], [40, 1, 1], [1, 0, 1]):
            T, most = sum(max(0, v) for v in add), max(add)
            log(f"step of {T} rows, at most {most} a request")
            want = plan_oracle(page, n_pages, rows, ln, np.array(add), table, ring, ctl)
            plan = Plan(page, n_pages, rows, ln, np.array(add), table, ring, ctl, in_place=True)
            s.conv, s.state = conv, state
            step = Step(layer, s, rows, most, plan)
            x, h = (rng.standard_normal((rows, HID)).astype(np.float32) for _ in range(2))
            step.feed(x, h, add)
            for c in step.calls():
                R.check(c(), "call")
            moe = Dev(nbytes=T * HID * 4, shape=(T, HID))
            R.check(R.lib().roaster_moe_prefill(table_moe.t, 0, step.y.p, T, moe.p, None) if T > 8 else
                    R.lib().roaster_moe_decode(table_moe.t, 0, step.y.p, T, moe.p, None), "moe")
            last = R.RoasterNorm(T, HID, HID, moe.p, HID, step.h.p, HID, None, None, 0, EPS, moe.p, HID, None, 0, None)
            held = step.h
            sync()
            g = step.got()
            for name, value in want.items():
                assert np.array_equal(g[name], value), name
            out = check_step(layer, g, x, h, T, s, [max(0, v) for v in add], ln, conv, state)
            assert np.all(g["mix"][T:] == 77)
            m = moe.get()
            assert np.isfinite(m).all()
            R.check(R.lib().roaster_norm(C.byref(last)), "norm")
            sync()
            after = held.get()[:T]
            assert np.array_equal(after, g["h"][:T] + m)
            y = norm_oracle(after, HID, None, None, EPS)
            assert np.all(np.abs(moe.get() - y) <= REL * np.abs(y) + 1e-37)
            log(f"  scan's out and state use {out[0]:.2g} and {out[1]:.2g} of their bounds")
            conv, state = g["conv"], g["state"]
            ln, table, ring, ctl = g["len_out"], g["table"], g["ring"], g["ctl_out"]
    finally:
        table_moe.destroy()


ADDS = [(12, 6, 5, [[1] * 6, [1, 1, 0, 1, -1, 1], [2, 2, 2, 2, 2, 2], [0] * 6, [5, 0, 1, 0, 3, 0]]),
        (90, 4, 80, [[20, 3, 10, 7], [1, 1, 1, 1], [0, 80, 0, 0], [30, -1, 33, 1], [0, 0, 0, 0], [2, 70, 1, 0]])]


@pytest.mark.parametrize("rows,n,most,adds", ADDS)
def test_captured_step(layer, rows, n, most, adds):
    """A step captured once and replayed with other lengths each time, its rows padded: every replay equal, bit for bit, to the
    same calls made eagerly on a state of their own, with eager work of the library between the replays."""
    rng = np.random.default_rng(rows)
    R.check(R.lib().roaster_init(), "init")
    start = np.array([33, 0, 100, 16, 5, 64][:n], np.int32)
    s = Scan(rng, [1] * n, [0] * n, R.SCAN_DELTA, KH, VH, KD, VD, TAPS)
    n_pages, table, ring, ctl = pool(rng, 16, start, 40, 16)
    sides = [Step(layer, s, rows, most, Plan(16, n_pages, rows, start, np.zeros(n, np.int32), table, ring, ctl, in_place=True)) for _ in range(2)]
    a, b = sides
    g = Graph(a.calls())
    try:
        ln, conv, state = start, s.conv, s.state
        for i, add in enumerate(adds):
            log(f"replay {i} of {rows} rows: adds {add}")
            x, h = (rng.standard_normal((rows, HID)).astype(np.float32) for _ in range(2))
            for side in sides:
                side.feed(x, h, add)
            g.launch()
            sync()
            for c in b.calls():
                R.check(c(), "call")
            sync()
            want, got = b.got(), a.got()
            for name, value in got.items():
                assert np.array_equal(value.view(np.uint8), want[name].view(np.uint8)), (i, name)
            T = sum(max(0, v) for v in add)
            if T:
                check_step(layer, want, x, h, T, s, [max(0, v) for v in add], ln, conv, state)
            ln, conv, state = want["len_out"], want["conv"], want["state"]
    finally:
        g.destroy()


def test_two_graphs_with_states_of_their_own_beside_each_other(layer):
    """Two captured steps replayed on two streams at once, each with its own buffers, against the same steps made eagerly."""
    import torch
    R.check(R.lib().roaster_init(), "init")
    sides = []
    for i, (rows, most, add) in enumerate(((64, 40, [30, 20]), (3, 1, [1, 1, 1]))):
        rng, n = np.random.default_rng(50 + i), len(add)
        start = np.array([5, 0, 9][:n], np.int32)
        s = Scan(rng, [1] * n, [0] * n, R.SCAN_DELTA, KH, VH, KD, VD, TAPS)
        n_pages, table, ring, ctl = pool(rng, 16, start, 40, 16)
        x, h = (rng.standard_normal((rows, HID)).astype(np.float32) for _ in range(2))

        def make():
            step = Step(layer, s, rows, most, Plan(16, n_pages, rows, start, np.zeros(n, np.int32), table, ring, ctl, in_place=True))
            step.feed(x, h, add)
            return step

        a, b = make(), make()
        sides.append((a, b, Graph(a.calls()), torch.cuda.Stream()))
    try:
        for rep in range(4):
            sync()
            for _, _, g, stream in sides:
                assert Graph.hip.hipGraphLaunch(g.run_it, C.c_void_p(stream.cuda_stream)) == 0
            torch.cuda.synchronize()
            for _, b, _, _ in sides:
                for c in b.calls():
                    R.check(c(), "call")
            sync()
            for a, b, _, _ in sides:
                want = b.got()
                for name, value in a.got().items():
                    assert np.array_equal(value.view(np.uint8), want[name].view(np.uint8)), (rep, name)
    finally:
        for _, _, g, _ in sides:
            g.destroy()


def test_errors_of_several_calls_are_reported_one_by_one(layer):
    """A plan without pages, a bad row of attention and a bad position of the scan before one sync."""
    from test_gpu_attn import make
    rng = np.random.default_rng(4)
    L = R.lib()
    n_pages, table, ring, ctl = pool(rng, 16, np.array([16]), 0, 4, slack=0)
    few = Plan(16, n_pages, 8, [16], [3], table, ring, ctl)
    kc, vc, table = make(rng, [20], 2, 64, 16, True)
    attn = Attn(Cache(kc, vc), np.zeros((1, 4, 64), np.float32), np.array([5], np.int32), np.array([3], np.int32), table, 1.0)
    scan = ScanCall(Scan(rng, [2], [-3], R.SCAN_STATE, 1, 1, 64, 64))
    for calls, codes in (([scan, few, attn], [R.ENOMEM, R.EINVAL, R.EINVAL]), ([scan, scan], [R.EINVAL]), ([scan, attn], [R.EINVAL, R.EINVAL])):
        for c in calls:
            R.check(c.call(), "call")
        said = []
        for code in codes:
            assert L.roaster_sync() == code, (codes, said)
            said.append(R.last_error())
        assert len(set(said)) == len(codes) and "left out" in said[-1]
        assert L.roaster_sync() == R.OK
