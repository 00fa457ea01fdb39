"""roaster_norm against the formulas in 64 bits.

The residual's sum is one f32 addition and compared bit by bit.  Bound of an element of
y, relative: the mean of squares of a row of 4 V L elements is off by at most 4 V + 12
roundings and halves its own in the root; root, division, product with the weight and
with the gate, whose sigmoid takes an exponential, an addition and a division: 12 more.
V is at most 16.  Values in 8 bits are those of the f32 output, bit by bit, where both are asked for;
alone they are off by half a step and 127 times the bound more."""
import ctypes as C

import numpy as np
import pytest

import roaster_amd as R
from attn_util import EPS24, sync
from gpu_util import Dev
from mixer_util import eights, norm_oracle

pytestmark = pytest.mark.gpu
EPS = 1e-6
REL = ((4 * 16 + 12) / 2 + 12) * EPS24


class Norm:
    def __init__(self, x, group, res=None, weight=None, gate=None, y=True, q=False, pad=0, in_place=False, eps=EPS, cols=None):
        T, D = x.shape[0], cols or x.shape[1]
        self.d = {k: Dev(v) if v is not None else None for k, v in dict(x=x, res=res, weight=weight, gate=gate).items()}
        self.y = (self.d["x"] if in_place else Dev(np.full((T, D + pad), 77, np.float32))) if y else None
        self.q = Dev(np.full((T, D + pad), 77, np.int8)) if q else None
        self.scale = Dev(np.full(T, 77, np.float32)) if q else None
        p = lambda b: b.p if b else None  # noqa: E731
        width = lambda v: v.shape[1] if v is not None else 0  # noqa: E731
        self.a = R.RoasterNorm(T, D, group, p(self.d["x"]), width(x), p(self.d["res"]), width(res), p(self.d["weight"]),
                               p(self.d["gate"]), width(gate), eps, p(self.y), x.shape[1] if in_place else D + pad, p(self.q), D + pad,
                               p(self.scale))

    def call(self):
        return R.lib().roaster_norm(C.byref(self.a))


def near(got, want):
    err = np.abs(got.astype(np.float64) - want)
    lim = REL * np.abs(want) + 1e-37
    assert np.all(err <= lim), float((err / lim).max())


@pytest.mark.parametrize("T,D,group", [
    (1, 2048, -1), (1, 4, -1), (3, 20, -1), (2, 60, -1), (5, 1028, -1), (7, 2052, -1), (2, 4096, -1), (3, 8196, -1), (2, 16384, -1),
    (900, 2048, -1), (1500, 500, -1), (700, 4096, 128), (1, 4096, 128), (3, 2048, 256), (5, 96, 16), (4, 16384, 64), (6, 320, 32), (3, 64, 64), (2, 128, 0),
    (1300, 72, -1), (2048, 4096, 128)])
@pytest.mark.parametrize("res,gate,q", [(1, 0, 0), (0, 1, 2), (1, 1, 1), (0, 0, 2)])
def test_norm(T, D, group, res, gate, q):
    rng = np.random.default_rng(T + D + group)
    pad = 4 * (D % 3)
    group = D if group < 0 else group
    x, r, g = (rng.standard_normal((T, D + 4 * i)).astype(np.float32) * np.float32(s) for i, s in ((1, 3), (2, 1), (0, 4)))
    w = (1 + 0.3 * rng.standard_normal(max(4, group))).astype(np.float32) if group and T % 2 else None
    n = Norm(x, group, r if res else None, w, g if gate else None, y=q != 1, q=q > 0, pad=pad, cols=D)
    R.check(n.call(), "norm")
    sync()
    v = x[:, :D]
    if res:
        v = v + r[:, :D]
        got = n.d["res"].get()
        assert np.array_equal(got[:, :D], v) and np.array_equal(got[:, D:], r[:, D:])
    want = norm_oracle(v, group, w, g if gate else None, EPS)
    if q != 1:
        y = n.y.get()
        near(y[:, :D], want)
        assert np.all(y[:, D:] == 77)
    if q:
        k, s = n.q.get(), n.scale.get()
        assert np.all(k[:, D:] == 77)
        if q == 2:
            kk, ss = eights(y[:, :D])
            assert np.array_equal(k[:, :D], kk) and np.array_equal(s, ss)
        top = np.abs(want).max(axis=1)
        assert np.all(np.abs(s - top / 127) <= (REL + 2 * EPS24) * top / 127 + 1e-37)
        assert np.all(np.abs(k[:, :D] * s[:, None].astype(np.float64) - want) <= (0.5 + 127 * (2 * REL + 4 * EPS24)) * s[:, None])


def test_in_place_and_a_row_for_all():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((9, 512)).astype(np.float32)
    r = rng.standard_normal((9, 512)).astype(np.float32)
    n = Norm(x, 512, r, in_place=True)
    R.check(n.call(), "norm")
    sync()
    near(n.y.get(), norm_oracle(x + r, 512, None, None, EPS))
    n = Norm(x, 64, r)
    n.a.x_row = 0
    R.check(n.call(), "norm")
    sync()
    assert np.array_equal(n.d["res"].get(), x[:1] + r)
    near(n.y.get(), norm_oracle(x[:1] + r, 64, None, None, EPS))


@pytest.mark.parametrize("D,group", [(256, 256), (2052, 2052), (512, 64)])
def test_odd_values(D, group):
    """Zeros, the smallest and largest numbers, infinities and NaN: each row by itself, and a row of heads head by head."""
    rng = np.random.default_rng(D)
    x = rng.standard_normal((8, D)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(1e-30)
    x[2] = np.float32(2.0 ** -149)
    x[3, 5] = np.inf
    x[4, 7] = np.nan
    x[5] *= np.float32(1e15)
    g = np.ones((8, D), np.float32)
    g[6, 3], g[6, 4] = 200, -200
    n = Norm(x, group, gate=g, q=True, eps=1e-30)
    R.check(n.call(), "norm")
    sync()
    y, k, s = n.y.get(), n.q.get(), n.scale.get()
    with np.errstate(all="ignore"):
        want = norm_oracle(x, group, None, g, 1e-30)
    assert not y[0].any() and not k[0].any() and s[0] == 0
    for r in (1, 2, 5, 6, 7):
        near(y[r], want[r])
        kk, ss = eights(y[r:r + 1])
        assert np.array_equal(k[r], kk[0]) and s[r] == ss[0]
    for r, c in ((3, 5), (4, 7)):
        head = slice(c // group * group, (c // group + 1) * group)
        rest = np.ones(D, bool)
        rest[head] = False
        assert np.isnan(y[r, c]) and np.isfinite(y[r, rest]).all()
        near(y[r, rest], want[r, rest])
        assert np.isnan(s[r]) and not k[r].any()
    # a row too small for a scale
    n = Norm(np.full((2, 64), 2.0 ** -125, np.float32), 0, q=True)
    R.check(n.call(), "norm")
    sync()
    assert not n.q.get().any() and not n.scale.get().any() and np.all(n.y.get() == 2.0 ** -125)


@pytest.mark.parametrize("D,group", [(256, 256), (512, 64)])
def test_rows_whose_squares_pass_the_range_are_zeros(D, group):
    """The residual is added all the same; other rows, and a row's other heads, come out as without it."""
    rng = np.random.default_rng(D + 1)
    x, r = (rng.standard_normal((4, D)).astype(np.float32) for _ in range(2))
    x[1, :group] = np.float32(3e19)
    n = Norm(x, group, r, q=True)
    R.check(n.call(), "norm")
    sync()
    v = x + r
    assert np.array_equal(n.d["res"].get(), v)
    y, k, s = n.y.get(), n.q.get(), n.scale.get()
    fine = np.ones((4, D), bool)
    fine[1, :group] = False
    with np.errstate(over="ignore"):
        want = norm_oracle(v, group, None, None, EPS)
    near(y[fine], want[fine])
    assert not y[~fine].any() and not k[~fine].any()
    kk, ss = eights(y)
    assert np.array_equal(k, kk) and np.array_equal(s, ss)
