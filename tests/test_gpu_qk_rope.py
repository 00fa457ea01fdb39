"""roaster_qk_rope_store against the formulas in 64 bits.

Bound of an f32 element: its pair's sum of sizes times 20 roundings of 2^-24
(the mean of squares halves its own 12, then the root, the division, two
products, the angle's cos and sin at 2 each, the rotation's two); an fp16 one
half a step (2^-11, or 2^-25 below the normal range) more."""
import ctypes as C

import numpy as np
import pytest

import roaster_amd as R
from attn_util import EPS24, Cache, rope_oracle, sync
from gpu_util import Dev, log

pytestmark = pytest.mark.gpu
EPS, THETA = 1e-6, 1e7


def near(got, want, size, f16):
    lim = size * 20 * EPS24 + (np.maximum(np.abs(want) * 2.0 ** -11, 2.0 ** -25) if f16 else 0) + 1e-30
    err = np.abs(got.astype(np.float64) - want)
    assert np.all(err <= lim), float((err / lim).max())


def run_case(T, H, KV, D, rot, f16, page=16, adjacent=0, norm=True, far=5000, gap=0, gated=True, in_place=False, skip=(),
             eps=EPS, theta=THETA, seed=0, pos=None):
    rng = np.random.default_rng(seed * 1000 + T + H + D + rot)
    per = 2 if gated and not in_place else 1
    q = (3 * rng.standard_normal((T, H, per, D))).astype(np.float32)
    k = (2 * rng.standard_normal((T, KV + gap, D))).astype(np.float32)       # `gap` heads between the rows are not this call's
    v = rng.standard_normal((T, KV, D + 4 * gap)).astype(np.float32)
    qn, kn = ((1 + 0.3 * rng.standard_normal((2, D))).astype(np.float32) if norm else (None, None))
    pos = rng.integers(0, far, T).astype(np.int32) if pos is None else np.asarray(pos, np.int32)
    n_pages = -(-2 * T // page) + 1
    slot = rng.permutation(n_pages * page)[:T].astype(np.int32)
    for t in skip:
        slot[t] = -1
    dt = np.float16 if f16 else np.float32
    kc, vc = (rng.standard_normal((n_pages, KV, page, D)).astype(dt) for _ in range(2))
    c = Cache(kc, vc)
    dq, dk, dv, dp, ds = (Dev(a) for a in (q, k, v, pos, slot))
    dqn, dkn = (Dev(a) if a is not None else None for a in (qn, kn))
    out = dq if in_place else Dev(np.full((T, H, D), 77, np.float32))
    a = R.RoasterQkRope(T, H, dq.p, per * H * D, per * D, dk.p, (KV + gap) * D, D, dv.p, KV * (D + 4 * gap), D + 4 * gap,
                        dqn.p if norm else None, dkn.p if norm else None, eps, rot, adjacent, theta, dp.p, ds.p, out.p)
    R.check(R.lib().roaster_qk_rope_store(C.byref(a), C.byref(c.c)), "rope")
    sync()
    live = slot >= 0
    want, size = rope_oracle(q[:, :, 0], qn, pos, eps, rot, adjacent, theta)
    got = out.get().reshape(T, H, D)
    near(got[live], want[live], size[live], False)
    assert np.array_equal(got[~live], q[~live][:, :, 0] if in_place else np.full_like(got[~live], 77))
    want, size = rope_oracle(k[:, :KV], kn, pos, eps, rot, adjacent, theta)
    gk, gv = c.k.get(), c.v.get()
    pg, at = slot[live] // page, slot[live] % page
    near(gk[pg, :, at], want[live], size[live], f16)
    assert np.array_equal(gv[pg, :, at], v[live][:, :, :D].astype(dt))
    kc[pg, :, at], vc[pg, :, at] = gk[pg, :, at], gv[pg, :, at]
    assert np.array_equal(gk, kc) and np.array_equal(gv, vc)                  # and nothing else is written


HEADS = [(16, 2, 256, 64), (16, 2, 256, 256), (1, 1, 256, 8), (32, 8, 128, 128), (7, 1, 128, 40), (20, 4, 64, 64),
         (9, 3, 64, 24), (5, 5, 64, 0)]


@pytest.mark.parametrize("H,KV,D,rot", HEADS)
@pytest.mark.parametrize("adjacent", [0, 1])
@pytest.mark.parametrize("f16", [True, False])
def test_heads(H, KV, D, rot, adjacent, f16):
    log(f"rope H={H} KV={KV} D={D} rot={rot} adjacent={adjacent} f16={f16}")
    for T, page in ((1, 16), (5, 64), (37, 16)):
        run_case(T, H, KV, D, rot, f16, page=page, adjacent=adjacent, seed=T)


@pytest.mark.parametrize("T", [511, 767, 768, 1100])
def test_many_rows(T):
    run_case(T, 16, 2, 256, 64, True, page=64, skip=(0, 3, T - 1))
    run_case(T, 20, 4, 64, 64, False, page=32, skip=(7,))


def test_strides_and_no_norm():
    run_case(6, 8, 2, 128, 64, True, gap=3, norm=False)
    run_case(6, 8, 2, 128, 64, False, gap=1, gated=False)


@pytest.mark.parametrize("H,KV,D,rot", HEADS[:3] + HEADS[5:6])
def test_queries_in_place(H, KV, D, rot):
    run_case(33, H, KV, D, rot, True, in_place=True, skip=(4, 5))
    run_case(700, H, KV, D, rot, True, in_place=True, skip=(4, 5))


def test_far_positions():
    """Up to the last position an int holds: in 32 bits the angle itself would be lost."""
    pos = [0, 1, 65535, 10 ** 6, 2 ** 24 + 1, 10 ** 9 + 7, 2 ** 31 - 2, 2 ** 31 - 1]
    run_case(8, 16, 2, 256, 64, False, pos=pos)
    run_case(8, 16, 2, 256, 256, False, pos=pos, theta=10000.0, adjacent=1)


def test_rows_of_zeros_and_large_values():
    """A head of zeros stays zeros (eps), one whose squares pass f32 is what the formula gives in f32."""
    q = np.zeros((1, 1, 1, 64), np.float32)
    run_case(3, 1, 1, 64, 64, False, eps=1.0)
    c = Cache(np.zeros((1, 1, 16, 64), np.float32), np.zeros((1, 1, 16, 64), np.float32))
    w, kv = Dev(np.ones(64, np.float32)), Dev(np.full((1, 1, 64), 1e30, np.float32))
    dq, out = Dev(q), Dev(np.full((1, 1, 64), 7, np.float32))
    pos, slot = Dev(np.array([5], np.int32)), Dev(np.array([3], np.int32))
    a = R.RoasterQkRope(1, 1, dq.p, 64, 64, kv.p, 64, 64, kv.p, 64, 64, w.p, w.p, EPS, 64, 0, THETA, pos.p, slot.p, out.p)
    R.check(R.lib().roaster_qk_rope_store(C.byref(a), C.byref(c.c)), "rope")
    sync()
    assert not out.get().any() and not c.k.get().any() and np.all(c.v.get()[0, 0, 3] == np.float32(1e30))


def test_fp16_values_past_the_range_become_infinite():
    c = Cache(np.zeros((1, 1, 16, 64), np.float16), np.zeros((1, 1, 16, 64), np.float16))
    x = np.zeros((1, 1, 64), np.float32)
    x[0, 0, :5] = [65504, 65519.9, 65520, -1e6, np.nan]
    dx, out = Dev(x), Dev(np.zeros((1, 1, 64), np.float32))
    pos, slot = Dev(np.array([0], np.int32)), Dev(np.array([0], np.int32))
    a = R.RoasterQkRope(1, 1, dx.p, 64, 64, dx.p, 64, 64, dx.p, 64, 64, None, None, EPS, 0, 0, THETA, pos.p, slot.p, out.p)
    R.check(R.lib().roaster_qk_rope_store(C.byref(a), C.byref(c.c)), "rope")
    sync()
    with np.errstate(over="ignore"):
        assert np.array_equal(c.k.get()[0, 0, 0], x[0, 0].astype(np.float16), equal_nan=True)
        assert np.array_equal(c.v.get()[0, 0, 0], x[0, 0].astype(np.float16), equal_nan=True)


def test_slots_past_the_cache_are_reported_and_skipped():
    rng = np.random.default_rng(1)
    kc, vc = (rng.standard_normal((2, 2, 16, 128)).astype(np.float32) for _ in range(2))
    c = Cache(kc, vc)
    x = rng.standard_normal((4, 4, 128)).astype(np.float32)
    dx, out = Dev(x), Dev(np.full((4, 4, 128), 77, np.float32))
    pos, slot = Dev(np.arange(4, dtype=np.int32)), Dev(np.array([32, -1, 2 ** 31 - 1, -2 ** 31], np.int32))
    a = R.RoasterQkRope(4, 4, dx.p, 512, 128, dx.p, 512, 128, dx.p, 512, 128, None, None, EPS, 64, 0, THETA, pos.p, slot.p,
                        out.p)
    R.check(R.lib().roaster_qk_rope_store(C.byref(a), C.byref(c.c)), "rope")
    assert R.lib().roaster_sync() == R.EINVAL
    sync()
    assert np.array_equal(c.k.get(), kc) and np.array_equal(c.v.get(), vc) and np.all(out.get() == 77)
