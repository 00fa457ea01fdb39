"""Rows and states of a recurrent layer's operators that lie more than 2^32 bytes behind their tensor's start."""
import ctypes as C

import numpy as np
import pytest

import roaster_amd as R
from attn_util import EPS24, sync
from gpu_util import Dev, log
from mixer_util import Scan, ScanCall, check_scan, norm_oracle, packed, scan_oracle
from test_gpu_norm import REL

pytestmark = pytest.mark.gpu
FAR = 1 << 28                                               # elements between rows


class Rows:
    """Rows of a host array at a stride of FAR elements, at the end of a buffer as large as they need."""

    def __init__(self, rows, cols, dtype):
        self.shape, self.size, self.dtype = (rows, cols), np.dtype(dtype).itemsize, dtype
        self.p = R.lib().roaster_dev_alloc(((rows - 1) * FAR + cols) * self.size)
        assert self.p, R.last_error()

    def put(self, a):
        for r in range(self.shape[0]):
            row = np.ascontiguousarray(a[r])
            R.check(R.lib().roaster_h2d(self.p + r * FAR * self.size, row.ctypes.data, row.nbytes), "h2d")
        return self

    def get(self):
        out = np.empty(self.shape, self.dtype)
        for r in range(self.shape[0]):
            R.check(R.lib().roaster_d2h(out[r:].ctypes.data, self.p + r * FAR * self.size, self.shape[1] * self.size), "d2h")
        return out

    def free(self):
        R.lib().roaster_dev_free(self.p)


def test_norm():
    rng = np.random.default_rng(61)
    rows, cols = 6, 256
    x, res = (rng.standard_normal((rows, cols)).astype(np.float32) for _ in range(2))
    dx, dr, dy = Rows(rows, cols, np.float32).put(x), Rows(rows, cols, np.float32).put(res), Rows(rows, cols, np.float32)
    try:
        a = R.RoasterNorm(rows, cols, cols, dx.p, FAR, dr.p, FAR, None, None, 0, 1e-6, dy.p, FAR, None, 0, None)
        R.check(R.lib().roaster_norm(C.byref(a)), "norm")
        sync()
        assert np.array_equal(dr.get(), res + x)
        want = norm_oracle(res + x, cols, None, None, 1e-6)
        assert np.all(np.abs(dy.get() - want) <= REL * np.abs(want) + 1e-37)
    finally:
        for d in (dx, dr, dy):
            d.free()


@pytest.mark.parametrize("T", [18, 40])
def test_matmul(T):
    rng = np.random.default_rng(62)
    N, K = 48, 160
    xq, wq = rng.integers(-128, 128, (T, K)).astype(np.int8), rng.integers(-128, 128, (N, K)).astype(np.int8)
    xs, ws = rng.uniform(0.01, 0.1, T).astype(np.float32), rng.uniform(0.01, 0.1, N).astype(np.float32)
    dx, dy = Rows(T, K, np.int8).put(xq), Rows(T, N, np.float32)
    dw, dxs, dws = Dev(packed(wq)), Dev(xs), Dev(ws)
    try:
        w = R.RoasterI8(dw.p, dws.p, N, K)
        a = R.RoasterMatmulI8(T, dx.p, FAR, dxs.p, dy.p, FAR)
        R.check(R.lib().roaster_matmul_i8(C.byref(a), C.byref(w)), "matmul_i8")
        sync()
        want = (xq.astype(np.float64) @ wq.astype(np.float64).T) * xs[:, None].astype(np.float64) * ws.astype(np.float64)
        assert np.all(np.abs(dy.get() - want) <= 3 * EPS24 * 1.01 * np.abs(want))
    finally:
        dx.free()
        dy.free()


@pytest.mark.parametrize("new", [[1] * 18, [18], [5, 13]])
def test_scan_rows(new):
    """18 rows: single tokens, by chunks, a few tokens each."""
    rng = np.random.default_rng(63)
    s = Scan(rng, new, [3] * len(new), R.SCAN_DELTA, 1, 2, 64, 64)
    T = s.rows
    d = [Rows(T, s.C, np.float32).put(s.x), Rows(T, s.vh, np.float32).put(s.a), Rows(T, s.vh, np.float32).put(s.b),
         Rows(T, s.vh * s.vd, np.float32)]
    try:
        c = ScanCall(s, x=d[0].p, x_row=FAR, a=d[1].p, a_row=FAR, b=d[2].p, b_row=FAR, out=d[3].p, out_row=FAR)
        R.check(c.call(), "scan")
        sync()
        out = d[3].get().reshape(T, s.vh, s.vd)
        log(check_scan((out, c.d["conv"].get(), c.d["state"].get()), scan_oracle(s)))
    finally:
        for v in d:
            v.free()


@pytest.mark.parametrize("new", [1, 3, 50])
def test_scan_states(new):
    """2048 requests of 32 heads of 128 x 128: the last one's state begins 4.29 GB behind the first's."""
    rng = np.random.default_rng(64)
    n, last = 2048, 2047
    s = Scan(rng, [new], [7], R.SCAN_DELTA, 2, 32, 128, 128)
    L = R.lib()
    one, two = s.conv.nbytes, s.state.nbytes
    conv, state = L.roaster_dev_alloc(n * one), L.roaster_dev_alloc(n * two)
    assert conv and state, R.last_error()
    try:
        for base, size, a in ((conv, one, s.conv), (state, two, s.state)):
            R.check(L.roaster_h2d(base + last * size, a.ctypes.data, size), "h2d")
        first = Dev(np.array([0] * n + [new], np.int32))
        st = R.RoasterSsmState(n, s.kh, s.vh, s.kd, s.vd, s.taps, conv, state)
        need = L.roaster_ssm_ws_bytes(s.rows, new, C.byref(st))
        ws = Dev(np.full(need, 0xFF, np.uint8))
        c = ScanCall(s, first=first.p, ws=ws.p, ws_bytes=need)
        R.check(L.roaster_ssm_scan(C.byref(c.a), C.byref(st)), "scan")
        sync()
        got = [c.out.get(), np.empty_like(s.conv), np.empty_like(s.state)]
        for base, size, a in ((conv, one, got[1]), (state, two, got[2])):
            R.check(L.roaster_d2h(a.ctypes.data, base + last * size, size), "d2h")
        log(check_scan(got, scan_oracle(s)))
    finally:
        L.roaster_dev_free(conv)
        L.roaster_dev_free(state)
