"""roaster_ssm_scan against the recurrence in 64 bits, token by token (bounds: mixer_util.scan_oracle)."""
import numpy as np
import pytest

import roaster_amd as R
from attn_util import sync
from gpu_util import Dev, log
from mixer_util import Scan, ScanCall, check_scan, scan_oracle

pytestmark = pytest.mark.gpu
DELTA, STATE = R.SCAN_DELTA, R.SCAN_STATE


def run(s, **kw):
    c = ScanCall(s, **kw)
    R.check(c.call(), "scan")
    sync()
    return c.got()


SHAPES = [(2, 4, 128, 128), (3, 3, 64, 64), (1, 5, 128, 64), (2, 2, 64, 128)]


@pytest.mark.parametrize("kh,vh,kd,vd", SHAPES)
@pytest.mark.parametrize("mode", [DELTA, STATE])
@pytest.mark.parametrize("new,pos", [
    ([1], [0]), ([1, 0, 1, 1], [7, 3, 0, 2]), ([3], [0]), ([5, 1, 0, 2], [2, 1, 9, 0]), ([64], [0]), ([65], [5]), ([20, 70, 0, 130], [0, 11, 4, 3]),
    ([1, 2, 3, 33, 31], [1, 2, 3, 0, 1000000])])
def test_scan(kh, vh, kd, vd, mode, new, pos):
    rng = np.random.default_rng(sum(new) + kd + 2 * vd + mode)
    for taps in (2, 3, 4):
        s = Scan(rng, new, pos, mode, kh, vh, kd, vd, taps, pad=taps - 2, bias=taps != 3, dt_bias=taps != 2, skip=taps == 4, wide=taps - 2)
        o, st = check_scan(run(s), scan_oracle(s))
        log(f"taps {taps}: out {o:.2g}, state {st:.2g} of their bounds")


@pytest.mark.parametrize("mode", [DELTA, STATE])
def test_a_long_prompt(mode):
    s = Scan(np.random.default_rng(5), [700], [0], mode, 2, 4, 128, 128)
    log(check_scan(run(s), scan_oracle(s)))


@pytest.mark.parametrize("most", [6, 40, 200])
def test_a_larger_most_gives_the_same(most):
    """Requests of few tokens under bounds that allow more."""
    s = Scan(np.random.default_rng(9), [3, 1, 6, 0], [0, 5, 2, 8], DELTA, 2, 4, 128, 64, pad=190)
    check_scan(run(s, most=most), scan_oracle(s))


def test_the_same_call_gives_the_same_bits():
    s = Scan(np.random.default_rng(6), [90, 1, 40], [0, 3, 17], DELTA, 2, 4, 128, 128)
    a, b = run(s), run(s)
    assert all(np.array_equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("new", [[1, 1, 1], [9, 4, 2], [150, 40, 70]])
def test_a_first_token_starts_from_zeros(new):
    """NaN in the states of a request that begins, and of one without new tokens."""
    s = Scan(np.random.default_rng(8), new[:1] + [0] + new[1:], [0, 4, 3, 0], DELTA, 2, 2, 64, 64)
    want = scan_oracle(s)
    s.conv[0], s.state[0], s.conv[1], s.state[1], s.conv[3], s.state[3] = (np.nan,) * 6
    out, conv, state = run(s)
    for k, arr in ((1, conv), (2, state)):
        assert np.isnan(arr[1]).all()
        arr[1] = want[k][1]
    n = min(s.taps, new[0]), min(s.taps, new[2])
    for r, m in ((0, n[0]), (3, n[1])):                     # entries that no token has filled stay as they were
        conv[r, m:] = want[1][r, m:]
    check_scan((out, conv, state), want)


@pytest.mark.parametrize("mode", [DELTA, STATE])
@pytest.mark.parametrize("what", ["v", "k", "q", "a", "state"])
@pytest.mark.parametrize("new,at", [([1, 1, 1], 0), ([7, 9, 3], 4), ([130, 90, 20], 70)])
def test_infinities_and_nan_reach_only_what_uses_them(mode, what, new, at):
    """Request 1's row `at` holds a NaN or an infinity: the other requests, its rows before and the heads that
    do not use it come out as without it."""
    rng = np.random.default_rng(at + mode)
    s = Scan(rng, new, [3, 4, 0], mode, 2, 4, 64, 64, skip=False)
    want = scan_oracle(s)
    row = s.first[1] + at
    heads = range(2) if what in "kq" else range(1)
    for bad in (np.nan, np.inf):
        saved = {k: getattr(s, k).copy() for k in ("x", "a", "state")}
        if what == "v":
            s.x[row, 2 * 128 + 5] = bad
        elif what == "k":
            s.x[row, 128 + 9] = bad
        elif what == "q":
            s.x[row, 9] = bad
        elif what == "a":
            s.a[row, 0] = np.nan
        else:
            s.state[1, 0, 5, 3] = bad
        out, conv, state = run(s)
        assert not np.isfinite(out[row, 0, 5]) or what == "state" and at
        fine = np.ones(out.shape, bool)
        since = s.first[1] + (0 if what == "state" else at)
        for h in heads:
            if what in ("v", "state"):
                fine[since:s.first[2], h, 5] = False
            else:
                fine[since:s.first[2], h] = False
        lim = want[3] + 1e-30
        assert np.all(np.abs(out - want[0])[fine] <= lim[fine]), np.argwhere(fine & ~(np.abs(out - want[0]) <= lim))[:4].tolist()
        sf = np.ones(want[4].shape, bool)
        for h in heads:
            sf[1, h] = False
        if what in ("v", "state"):
            sf[1, 0] = True
            sf[1, 0, 5] = False
        es = np.linalg.norm(np.where(np.isfinite(state), state, 1e30) - want[2], axis=3)
        assert np.all(es[sf] <= want[4][sf] + 1e-30)
        for k, v in saved.items():
            setattr(s, k, v)


def test_bad_requests_are_left_out_and_reported():
    """Too many tokens, a negative position, rows out of range: the rows within are NaN, the states as they were,
    the others' results right, one report."""
    rng = np.random.default_rng(12)
    for most, pos, first in ((2, [0, 3, 5], None), (4, [0, -2, 5], None), (4, [0, 3, 5], [0, 2, 5, 70]), (4, [0, 3, 5], [0, 2, 1, 5]),
                             (40, [0, -7, 1], None)):
        big = most == 40
        new = [30, 36, 33] if big else [2, 3, 2]
        s = Scan(rng, new, pos, DELTA, 2, 2, 64, 64, pad=3)
        bad = 2 if first and first[3] == 70 else 1
        n = s.new[bad]
        s.new[bad] = 0
        want = scan_oracle(s)
        s.new[bad] = n
        if first:
            s.first = np.array(first, np.int32)
        c = ScanCall(s, most=most)
        R.check(c.call(), "scan")
        assert R.lib().roaster_sync() == R.EINVAL and "left out" in R.last_error()
        assert R.lib().roaster_sync() == R.OK
        out, conv, state = c.got()
        assert np.array_equal(conv[bad], s.conv[bad]) and np.array_equal(state[bad], s.state[bad])
        f = s.first
        if not first:
            assert np.isnan(out[f[1]:f[2]]).all()
        elif bad == 2:
            assert np.isnan(out[5:]).all()
        rows = slice(f[0], min(f[1], f[2]))                # a row that two requests claim is either's
        assert np.all(np.abs(out[rows] - want[0][rows]) <= want[3][rows] + 1e-30)
        if not first:
            rows = slice(f[2], None)
            assert np.all(np.abs(out[rows] - want[0][rows]) <= want[3][rows] + 1e-30)


def test_many_requests_mostly_idle():
    """2048 requests, a few with tokens."""
    rng = np.random.default_rng(15)
    new, pos = [0] * 2048, [1] * 2048
    for r, m in ((0, 1), (700, 3), (2047, 2)):
        new[r] = m
    s = Scan(rng, new, pos, STATE, 1, 1, 64, 64)
    check_scan(run(s), scan_oracle(s))
    new[5], new[1999] = 70, 40
    s = Scan(rng, new, pos, DELTA, 1, 1, 64, 64)
    check_scan(run(s), scan_oracle(s))


@pytest.mark.parametrize("qs,ks,scale", [(1, 1e22, 0.5), (1e22, 1, 0.5), (1e-24, 1, 1e22), (1, 1e-24, 1e22), (1e-24, 1e22, 3.0), (1e-30, 1e-30, 1e37)])
@pytest.mark.parametrize("new", [[2, 1], [70, 33]])
def test_vectors_whose_squares_leave_the_range(new, qs, ks, scale):
    """Without unit vectors only the vectors themselves have to be within f32's range."""
    s = Scan(np.random.default_rng(21), new, [0, 4], STATE, 1, 2, 128, 64, bias=False, skip=False, scale=scale)
    s.conv_w[:128] *= np.float32(qs)
    s.conv_w[128:256] *= np.float32(ks)
    s.state[1] *= np.float32(ks)
    out, conv, state = run(s)
    o, c, st, oe, se = scan_oracle(s)
    assert np.array_equal(conv.astype(np.float64), c)
    assert np.all(np.abs(out - o) <= oe)
    assert np.all(np.linalg.norm((state - st) / ks, axis=3) <= se / ks + 1e-9)       # that of -ks 1e-9: f32's least normal value


@pytest.mark.parametrize("new,at", [([2, 1], 1), ([70, 30], 5)])
def test_without_eps_a_zero_vector_is_nan_from_its_row_on(new, at):
    s = Scan(np.random.default_rng(22), new, [0, 4], DELTA, 2, 4, 128, 128, taps=2, bias=False)
    s.eps = 0.0
    want = scan_oracle(s)
    s.x[at - 1:at + 1, 256:384] = 0                         # key head 0's keys: value heads 0 and 1
    out, conv, state = run(s)
    bad = np.zeros(out.shape, bool)
    bad[at:new[0], :2] = True
    assert np.isnan(out[bad]).all() and np.isnan(state[0, :2]).all()
    ok = ~bad
    ok[at - 1] = False                                      # whose own key is another now
    assert np.all(np.abs(out - want[0])[ok] <= want[3][ok] + 1e-30)
    assert np.all(np.linalg.norm(state[1] - want[2][1], axis=2) <= want[4][1] + 1e-30)


@pytest.mark.parametrize("mode", [DELTA, STATE])
@pytest.mark.parametrize("new", [[3, 1], [100, 40]])
def test_decays_above_one(mode, new):
    s = Scan(np.random.default_rng(23), new, [0, 4], mode, 2, 4, 64, 128)
    s.a_coef = np.array([0.02, -0.5, 0.05, 0.0], np.float32)
    log(check_scan(run(s), scan_oracle(s)))


@pytest.mark.parametrize("noise", [0.0, 0.05])
def test_the_same_key_again_and_again(noise):
    """Gains of nearly one and hardly any decay: the solution takes back what the token before added."""
    s = Scan(np.random.default_rng(24), [200, 64], [0, 4], DELTA, 1, 2, 128, 64)
    keys = slice(128, 256)
    s.x[:, keys] = s.x[0, keys] + np.float32(noise) * s.x[:, keys]
    s.a[:], s.b[:] = -12, 8
    s.a_coef[:], s.dt_bias[:] = -0.1, 0
    log(check_scan(run(s), scan_oracle(s)))


@pytest.mark.parametrize("most", [15, 16, 23, 24, 31, 32, 39, 40])
@pytest.mark.parametrize("n", [1, 2, 40, 70])
def test_both_ways_about_their_limits(most, n):
    s = Scan(np.random.default_rng(most + n), [most] + [2] * (n - 1), [3] * n, DELTA, 2, 4, 128, 128)
    log(check_scan(run(s), scan_oracle(s)))


@pytest.mark.parametrize("mode", [DELTA, STATE])
@pytest.mark.parametrize("kd,vd", [(128, 64), (64, 128)])
@pytest.mark.parametrize("new", [[1] * 20 + [90] + [1] * 60 + [0, 200], [64, 1, 0, 23, 24, 25, 2, 65], [0, 1, 100], [1] * 130 + [30]])
def test_prompts_among_single_tokens(mode, kd, vd, new):
    rng = np.random.default_rng(len(new) + kd)
    pos = rng.integers(0, 5, len(new)).tolist()
    s = Scan(rng, new, pos, mode, 2, 2, kd, vd, pad=3)
    log(check_scan(run(s), scan_oracle(s)))


@pytest.mark.parametrize("new", [[2, 1], [70, 33]])
def test_a_wider_output(new):
    s = Scan(np.random.default_rng(26), new, [1, 0], DELTA, 1, 3, 64, 64, pad=2)
    c = ScanCall(s, out_row=3 * 64 + 12)
    c.out = Dev(np.full((s.rows, 3 * 64 + 12), 77, np.float32))
    c.a.out = c.out.p
    R.check(c.call(), "scan")
    sync()
    out, conv, state = c.got()
    assert np.all(out[:, 192:] == 77)
    check_scan((np.ascontiguousarray(out[:, :192]).reshape(s.rows, 3, 64), conv, state), scan_oracle(s))


@pytest.mark.parametrize("n", [4, 60])
def test_requests_that_share_rows(n):
    """More tokens than rows: a request whose chunks have no place left is reported and its state stays as it was."""
    s = Scan(np.random.default_rng(27), [640] + [0] * (n - 1), [2] + [0] * (n - 1), DELTA, 1, 1, 64, 64)
    want = scan_oracle(s)
    s.first = np.array([0, 640, 0, 640, 640] if n == 4 else [0, 640] + [0, 640] * 29 + [0], np.int32)
    c = ScanCall(s)
    R.check(c.call(), "scan")
    assert R.lib().roaster_sync() == R.EINVAL and "left out" in R.last_error()
    out, conv, state = c.got()
    # chunks of 64 rows, and one for each request that may have 24 rows of its own: of 14 chunks requests of ten find place once, of
    # 36 three times (every second one: those between are out of range)
    for r in [1, 2, 3] if n == 4 else [1, 3, 5] + list(range(6, n)):
        assert np.array_equal(state[r], s.state[r]) and np.array_equal(conv[r], s.conv[r])
    assert np.array_equal(conv[0].astype(np.float64), want[1][0])
    assert np.all(np.linalg.norm(state[0] - want[2][0], axis=2) <= want[4][0])


@pytest.mark.parametrize("n", [2, 40])
def test_rows_at_the_ends_of_an_int(n):
    """Differences of such rows do not fit an int: 2^31 - 1 to -2^31 would be one row."""
    s = Scan(np.random.default_rng(28), [n, 0, 0, 0], [3, 1, 2, 4], DELTA, 2, 2, 64, 64, pad=3)
    want = scan_oracle(s)
    s.first = np.array([0, n, 2 ** 31 - 1, -2 ** 31, 0], np.int64).astype(np.int32)
    c = ScanCall(s)
    R.check(c.call(), "scan")
    assert R.lib().roaster_sync() == R.EINVAL and "left out" in R.last_error()
    out, conv, state = c.got()
    assert np.all(np.abs(out[:n] - want[0][:n]) <= want[3][:n] + 1e-30) and np.isnan(out[n:]).all()
    assert np.array_equal(conv.astype(np.float64), want[1]) and np.array_equal(state[1:], s.state[1:])
    assert np.all(np.linalg.norm(state[0] - want[2][0], axis=2) <= want[4][0] + 1e-30)


@pytest.mark.parametrize("most", [39, 40, 47, 48])
@pytest.mark.parametrize("n,vh", [(70, 4), (33, 8)])
def test_both_ways_about_their_limits_with_64_keys(most, n, vh):
    s = Scan(np.random.default_rng(most + n), [most] + [2] * (n - 1), [3] * n, DELTA, 2, vh, 64, 64)
    log(check_scan(run(s), scan_oracle(s)))
