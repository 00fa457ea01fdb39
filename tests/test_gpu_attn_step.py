"""The attention operators as a serving step uses them together: plan, projections,
norms with rotation and store, attention, output projection, the MoE block -- each
step against 64-bit arithmetic on the host, and the steps of a captured graph
against the same calls made eagerly."""
import ctypes as C
import math

import numpy as np
import pytest

import roaster_amd as R
from attn_util import (Attn, Cache, EPS24, Plan, attn_oracle, check_attn, plan_oracle, pool, rope_oracle, sync)
from gpu_util import Dev, SynthTable, log, rel_err
from oracle import oracle as O

pytestmark = pytest.mark.gpu
H, KV, D, HID, ROT, PAGE = 16, 2, 256, 2048, 64, 32
EPS, THETA = 1e-6, 1e7


def weights(q6, rows, cols, stream):
    # entries of about 0.02, as a model's files have them
    n = rows * (cols // 256)
    return R.synth_q6k(5, stream, n, 3e-5, 9e-5) if q6 else R.synth_q4k(5, stream, n, 5e-5, 2e-4)


def project(w, q6, x, rows, cols):
    """roaster_matvec_q over rows of x, eight at a time."""
    y = Dev(nbytes=x.shape[0] * rows * 4, shape=(x.shape[0], rows))
    for t in range(0, x.shape[0], 8):
        T = min(8, x.shape[0] - t)
        R.check(R.lib().roaster_matvec_q(w.p, q6, x.p + t * cols * 4, y.p + t * rows * 4, rows, cols, T), "matvec_q")
    return y


@pytest.mark.parametrize("f16", [True, False])
def test_serving_steps_of_one_layer(f16):
    """Three requests: prompts of 5, 40 and 17 tokens, a step of one token each, a step in
    which the first ends, the second adds one and the third seven, and one more."""
    rng = np.random.default_rng(31)
    L = R.lib()
    host = [weights(0, 2 * H * D, HID, 1), weights(0, KV * D, HID, 2), weights(1, KV * D, HID, 3), weights(0, HID, H * D, 4)]
    wq, wk, wv, wo = (Dev(w) for w in host)
    qn, kn = ((1 + 0.2 * rng.standard_normal(D)).astype(np.float32) for _ in range(2))
    dqn, dkn = Dev(qn), Dev(kn)
    width, max_rows = 6, 70
    n_pages, table, ring, ctl = pool(rng, PAGE, np.zeros(3), 9, width, slack=0)
    dt = np.float16 if f16 else np.float32
    cache = Cache(*(np.full((n_pages, KV, PAGE, D), np.nan, dt) for _ in range(2)))
    ln, t_moe = np.zeros(3, np.int32), SynthTable(3, n_layers=1)
    try:
        for add in ([5, 40, 17], [1, 1, 1], [-1, 1, 7], [0, 1, 1]):
            add = np.array(add, np.int32)
            want = plan_oracle(PAGE, n_pages, max_rows, ln, add, table, ring, ctl)
            plan = Plan(PAGE, n_pages, max_rows, ln, add, table, ring, ctl, in_place=True)
            R.check(plan.call(), "plan")
            T = int(np.maximum(add, 0).sum())
            log(f"step of {T} rows, cache {'f16' if f16 else 'f32'}")
            x = rng.standard_normal((T, HID)).astype(np.float32)
            dx = Dev(x)
            q, k, v = project(wq, 0, dx, 2 * H * D, HID), project(wk, 0, dx, KV * D, HID), project(wv, 1, dx, KV * D, HID)
            qo = Dev(np.full((max_rows, H, D), 77, np.float32))
            rope = R.RoasterQkRope(T, H, q.p, 2 * H * D, 2 * D, k.p, KV * D, D, v.p, KV * D, D, dqn.p, dkn.p, EPS, ROT, 0, THETA,
                                   plan.row_pos.p, plan.row_slot.p, qo.p)
            R.check(L.roaster_qk_rope_store(C.byref(rope), C.byref(cache.c)), "rope")
            out = Dev(np.full((T, H, D), 77, np.float32))
            need = L.roaster_attn_ws_bytes(T, H, C.byref(cache.c))
            ws = Dev(nbytes=need)
            attn = R.RoasterAttnPaged(T, H, qo.p, plan.row_req.p, plan.row_pos.p, plan.table.p, 3, width, D ** -0.5,
                                      q.p + 4 * D, 2 * H * D, 2 * D, out.p, ws.p, need)
            R.check(L.roaster_attn_paged(C.byref(attn), C.byref(cache.c)), "attn")
            y = project(wo, 0, out, HID, H * D)
            moe = Dev(nbytes=T * HID * 4, shape=(T, HID))
            for t in range(0, T, 8):
                R.check(L.roaster_moe_decode(t_moe.t, 0, y.p + t * HID * 4, min(8, T - t), moe.p + t * HID * 4, None), "moe")
            sync()
            # the plan
            got = plan.got()
            for name, value in want.items():
                assert np.array_equal(got[name], value), name
            ln, table, ring, ctl = got["len_out"], got["table"], got["ring"], got["ctl_out"]
            req, pos, slot = (got[n][:T] for n in ("row_req", "row_pos", "row_slot"))
            # projections (sampled), norms and rotation, the cache
            pq, pk, pv = q.get(), k.get(), v.get()
            for t in (0, T - 1):
                assert rel_err(pq[t], O.matvec(0, host[0], x[t], 2 * H * D, HID)) <= 2e-5
                assert rel_err(pv[t], O.matvec(1, host[2], x[t], KV * D, HID)) <= 2e-5
            ref, size = rope_oracle(pq.reshape(T, H, 2, D)[:, :, 0], qn, pos, EPS, ROT, 0, THETA)
            rows = qo.get()
            assert np.all(np.abs(rows[:T] - ref) <= 20 * EPS24 * size + 1e-30) and np.all(rows[T:] == 77)
            kc, vc = cache.k.get(), cache.v.get()
            ref, size = rope_oracle(pk.reshape(T, KV, D), kn, pos, EPS, ROT, 0, THETA)
            lim = 20 * EPS24 * size + (np.abs(ref) * 2.0 ** -11 + 2.0 ** -25 if f16 else 0) + 1e-30
            assert np.all(np.abs(kc[slot // PAGE, :, slot % PAGE].astype(np.float64) - ref) <= lim)
            assert np.array_equal(vc[slot // PAGE, :, slot % PAGE], pv.reshape(T, KV, D).astype(dt))
            # attention from what the cache holds, the output projection from what attention gave
            a = out.get()
            rel = check_attn(a, *attn_oracle(rows[:T], kc, vc, table, req, pos, 0.0625, pq.reshape(T, H, 2, D)[:, :, 1]),
                             int(pos.max()) + 1, D)
            o = y.get()
            for t in (0, T - 1):
                assert rel_err(o[t], O.matvec(0, host[3], a[t].reshape(-1), HID, H * D)) <= 2e-5
            assert np.isfinite(moe.get()).all()
            log(f"  attention rel {rel:.1e}")
    finally:
        t_moe.destroy()


class Graph:
    """Calls captured from the library's stream."""

    hip = None

    def __init__(self, calls):
        if Graph.hip is None:
            Graph.hip = C.CDLL("libamdhip64.so")
        h, self.stream = Graph.hip, C.c_void_p(R.lib().roaster_stream())
        graph, self.run_it = C.c_void_p(), C.c_void_p()
        assert h.hipStreamBeginCapture(self.stream, 1) == 0            # thread-local
        rcs = [c() for c in calls]
        assert h.hipStreamEndCapture(self.stream, C.byref(graph)) == 0 and rcs == [0] * len(rcs)
        assert h.hipGraphInstantiate(C.byref(self.run_it), graph, None, None, C.c_size_t(0)) == 0
        assert h.hipGraphDestroy(graph) == 0

    def launch(self):
        assert Graph.hip.hipGraphLaunch(self.run_it, self.stream) == 0

    def destroy(self):
        assert Graph.hip.hipGraphExecDestroy(self.run_it) == 0


@pytest.mark.parametrize("rows,n,adds", [
    (12, 6, [[1] * 6, [1, 1, 0, 1, -1, 1], [2, 2, 2, 2, 2, 2], [0] * 6, [5, 0, 1, 0, 3, 0]]),
    (40, 4, [[20, 3, 10, 7], [1, 1, 1, 1], [0, 40, 0, 0], [30, -1, 1, 1], [0, 0, 0, 0]])])
@pytest.mark.parametrize("f16", [True, False])
def test_captured_step(rows, n, adds, f16):
    """A step captured once and replayed with other lengths each time, its rows padded: every
    replay equal, bit for bit, to the same calls made eagerly on a state of their own, with
    eager work of the library between the replays."""
    rng = np.random.default_rng(rows)
    L, page, width, heads, kv, dim = R.lib(), 16, 12, 8, 2, 128
    R.check(L.roaster_init(), "init")
    dt = np.float16 if f16 else np.float32
    start = np.array([33, 0, 100, 16, 5, 64][:n], np.int32)
    n_pages, table, ring, ctl = pool(rng, page, start, 40, width)
    kc, vc = (rng.standard_normal((n_pages, kv, page, dim)).astype(dt) for _ in range(2))
    x = [rng.standard_normal((rows, (heads + 2 * kv) * dim)).astype(np.float32) for _ in adds]

    class Side:
        def __init__(self):
            self.plan = Plan(page, n_pages, rows, start, np.zeros(n, np.int32), table, ring, ctl, in_place=True)
            self.cache, self.x = Cache(kc, vc), Dev(x[0])
            self.q = Dev(np.full((rows, heads, dim), 77, np.float32))
            p, row = self.x.p, (heads + 2 * kv) * dim
            self.rope = R.RoasterQkRope(rows, heads, p, row, dim, p + 4 * heads * dim, row, dim, p + 4 * (heads + kv) * dim,
                                        row, dim, None, None, EPS, 64, 1, 1e4, self.plan.row_pos.p, self.plan.row_slot.p,
                                        self.q.p)
            self.attn = Attn(self.cache, np.zeros((rows, heads, dim), np.float32), np.zeros(rows, np.int32),
                             np.zeros(rows, np.int32), table, dim ** -0.5)
            self.attn.a.q, self.attn.a.table = self.q.p, self.plan.table.p
            self.attn.a.row_req, self.attn.a.row_pos = self.plan.row_req.p, self.plan.row_pos.p

        def calls(self):
            return [self.plan.call, lambda: L.roaster_qk_rope_store(C.byref(self.rope), C.byref(self.cache.c)), self.attn.call]

        def feed(self, i):
            for d, a in ((self.plan.add, np.array(adds[i], np.int32)), (self.x, x[i])):
                R.check(L.roaster_h2d(d.p, a.ctypes.data, a.nbytes), "h2d")

        def got(self):
            return dict(self.plan.got(), q=self.q.get(), out=self.attn.out.get(), k=self.cache.k.get(), v=self.cache.v.get())

    a, b = Side(), Side()
    g = Graph(a.calls())
    try:
        for i in range(len(adds)):
            log(f"replay {i} of {rows} rows: adds {adds[i]}")
            for s in (a, b):
                s.feed(i)
            g.launch()
            sync()
            for c in b.calls():
                R.check(c(), "call")
            sync()
            want = b.got()
            for name, value in a.got().items():
                assert np.array_equal(value.view(np.uint8), want[name].view(np.uint8)), (i, name)
            used = sum(max(0, v) for v in adds[i])
            assert np.all(want["row_req"][used:] == -1)
            o = want["out"][:used]
            if used:
                check_attn(o, *attn_oracle(want["q"][:used], want["k"], want["v"], want["table"], want["row_req"][:used],
                                           want["row_pos"][:used], np.float64(np.float32(dim ** -0.5))),
                           int(want["row_pos"].max()) + 1, dim)
    finally:
        g.destroy()


def test_two_graphs_with_states_of_their_own_beside_each_other():
    """Two captured decode calls replayed on two streams at once, each with its own buffers."""
    import torch
    rng = np.random.default_rng(77)
    R.check(R.lib().roaster_init(), "init")
    from test_gpu_attn import make
    sides = []
    for i in range(2):
        kc, vc, table = make(rng, [700 + 900 * i, 65], 2, 256, 16, True)
        q = rng.standard_normal((2, 16, 256)).astype(np.float32)
        req, pos = np.array([0, 1], np.int32), np.array([699 + 900 * i, 64], np.int32)
        a = Attn(Cache(kc, vc), q, req, pos, table, 0.0625)
        sides.append((a, attn_oracle(q, kc, vc, table, req, pos, 0.0625), 700 + 900 * i, Graph([a.call]), torch.cuda.Stream()))
    try:
        for rep in range(5):
            for a, _, _, g, s in sides:
                R.check(R.lib().roaster_memset(a.out.p, 0, a.out.nbytes), "memset")
            sync()
            for _ in range(3):
                for _, _, _, g, s in sides:
                    assert Graph.hip.hipGraphLaunch(g.run_it, C.c_void_p(s.cuda_stream)) == 0
            torch.cuda.synchronize()
            for a, want, n, _, _ in sides:
                check_attn(a.out.get(), *want, n, 256)
    finally:
        for _, _, _, g, _ in sides:
            g.destroy()


def test_errors_wait_for_their_sync():
    """An attention error after a routing error is reported by the sync after that one's."""
    rng = np.random.default_rng(3)
    from test_gpu_attn import make
    L = R.lib()
    kc, vc, table = make(rng, [20], 2, 64, 16, True)
    a = Attn(Cache(kc, vc), np.zeros((1, 4, 64), np.float32), np.array([5], np.int32), np.array([3], np.int32), table, 1.0)
    t = SynthTable(3, n_layers=1)
    try:
        x, y = Dev(np.zeros((1, HID), np.float32)), Dev(np.zeros((1, HID), np.float32))
        lg = Dev(np.full((1, 256), -np.inf, np.float32))
        io = R.RoasterDecodeIO(lg.p, None, None, None)
        R.check(a.call(), "attn")
        R.check(L.roaster_moe_decode(t.t, 0, x.p, 1, y.p, C.byref(io)), "decode")
        assert L.roaster_sync() == R.EROUTE
        assert L.roaster_sync() == R.EINVAL
        assert L.roaster_sync() == R.OK
        assert math.isnan(a.out.get().ravel()[0])
    finally:
        t.destroy()


def test_errors_of_several_calls_are_reported_one_by_one():
    """A plan without pages, a plan whose lengths are out of range and a bad row before one sync:
    each is reported once, then none is left."""
    from test_gpu_attn import make
    rng = np.random.default_rng(4)
    L = R.lib()
    n_pages, table, ring, ctl = pool(rng, 16, np.array([16]), 0, 4, slack=0)
    few = Plan(16, n_pages, 8, [16], [3], table, ring, ctl)
    bad = Plan(16, n_pages, 8, [-4], [3], table, ring, ctl)
    kc, vc, table = make(rng, [20], 2, 64, 16, True)
    a = Attn(Cache(kc, vc), np.zeros((1, 4, 64), np.float32), np.array([5], np.int32), np.array([3], np.int32), table, 1.0)
    for calls, codes in (([few.call, a.call], [R.ENOMEM, R.EINVAL]), ([a.call, bad.call, few.call], [R.ENOMEM, R.EINVAL, R.EINVAL]),
                         ([a.call, a.call], [R.EINVAL]), ([bad.call, a.call], [R.EINVAL, R.EINVAL])):
        for c in calls:
            R.check(c(), "call")
        said = []
        for code in codes:
            assert L.roaster_sync() == code, (codes, said)
            said.append(R.last_error())
        assert len(set(said)) == len(codes)
        assert L.roaster_sync() == R.OK
