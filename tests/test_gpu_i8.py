"""roaster_i8_pack and roaster_matmul_i8.

The sums are whole numbers, so an element is off by the rounding of the sum to f32, of the two scales' product and of the product
with it: three halves of a step.  Packed values are compared with their definition in f32, bit by bit."""
import ctypes as C

import numpy as np
import pytest

import roaster_amd as R
from attn_util import EPS24, sync
from gpu_util import Dev
from mixer_util import eights, packed, unpacked
from oracle import oracle as O

pytestmark = pytest.mark.gpu


def matmul(xq, xs, wq, ws, x_pad=0, y_pad=0):
    T, K = xq.shape
    N = wq.shape[0]
    x = Dev(np.concatenate([xq, np.full((T, x_pad), 99, np.int8)], axis=1)) if x_pad else Dev(xq)
    dxs, dws, dw = Dev(xs), Dev(ws), Dev(packed(wq))
    y = Dev(np.full((T, N + y_pad), 77, np.float32))
    w = R.RoasterI8(dw.p, dws.p, N, K)
    a = R.RoasterMatmulI8(T, x.p, K + x_pad, dxs.p, y.p, N + y_pad)
    R.check(R.lib().roaster_matmul_i8(C.byref(a), C.byref(w)), "matmul_i8")
    sync()
    got = y.get()
    assert np.all(got[:, N:] == 77)
    return got[:, :N]


def values(rng, rows, cols):
    q = rng.integers(-128, 128, (rows, cols)).astype(np.int8)
    return q, rng.uniform(0.001, 0.1, rows).astype(np.float32)


def check(got, xq, xs, wq, ws):
    want = (xq.astype(np.float64) @ wq.astype(np.float64).T) * xs[:, None].astype(np.float64) * ws.astype(np.float64)
    assert np.all(np.abs(got - want) <= 3 * EPS24 * 1.01 * np.abs(want)), float((np.abs(got - want) / (EPS24 * np.abs(want) + 1e-300)).max())


@pytest.mark.parametrize("T", [1, 2, 8, 31, 32, 33, 64, 65, 100, 129, 257])
@pytest.mark.parametrize("N,K", [(1, 16), (33, 48), (64, 128), (100, 272), (257, 1040), (1000, 2064), (300, 4096)])
def test_matmul(T, N, K):
    rng = np.random.default_rng(T * 7 + N + K)
    (xq, xs), (wq, ws) = values(rng, T, K), values(rng, N, K)
    check(matmul(xq, xs, wq, ws, x_pad=16 * (T % 3), y_pad=N % 4), xq, xs, wq, ws)


@pytest.mark.parametrize("T,N,K", [(300, 12288, 512), (2048, 4096, 272), (700, 8192, 128), (520, 2500, 1024), (1, 20000, 256), (20, 9000, 2048),
                                   (130, 16000, 64), (1000, 1056, 160)])
def test_matmul_large(T, N, K):
    rng = np.random.default_rng(T + N + K)
    (xq, xs), (wq, ws) = values(rng, T, K), values(rng, N, K)
    check(matmul(xq, xs, wq, ws), xq, xs, wq, ws)


@pytest.mark.parametrize("T", [3, 70])
def test_largest_sums(T):
    """Every product at its largest over the longest rows: 2^30."""
    K, N = 65536, 40
    xq, wq = np.full((T, K), -128, np.int8), np.full((N, K), -128, np.int8)
    wq[1::2] = 127
    one = np.ones(T, np.float32), np.ones(N, np.float32)
    got = matmul(xq, one[0], wq, one[1])
    assert np.all(got[:, ::2] == 2.0 ** 30) and np.all(got[:, 1::2] == -128 * 127 * 65536.0)


@pytest.mark.parametrize("T", [5, 150])
def test_odd_scales_stay_in_their_rows(T):
    rng = np.random.default_rng(T)
    (xq, xs), (wq, ws) = values(rng, T, 64), values(rng, 70, 64)
    xs[2], xs[4], ws[11], ws[69] = np.nan, np.inf, np.nan, 0
    got = matmul(xq, xs, wq, ws)
    rows, cols = np.ones(T, bool), np.ones(70, bool)
    rows[[2, 4]], cols[11] = False, False
    assert np.isnan(got[2]).all() and np.isnan(got[:, 11]).all() and not np.isfinite(got[4]).any() and not got[rows][:, 69].any()
    check(got[rows][:, cols], xq[rows], xs[rows], wq[cols], ws[cols])


@pytest.mark.parametrize("rows,cols", [(1, 16), (33, 144), (70, 2064), (256, 256), (5, 65536)])
def test_pack_f32_and_i8(rows, cols):
    rng = np.random.default_rng(rows + cols)
    w = rng.standard_normal((rows, cols)).astype(np.float32)
    if rows > 4:
        w[1], w[2] = 0, np.float32(2.0 ** -130)
    n = R.lib().roaster_i8_bytes(rows, cols)
    dw, data, scale = Dev(w), Dev(np.full(n, 0x55, np.uint8)), Dev(np.full(rows, 77, np.float32))
    to = R.RoasterI8(data.p, scale.p, rows, cols)
    R.check(R.lib().roaster_i8_pack(dw.p, R.I8_FROM_F32, C.byref(to)), "pack")
    sync()
    q, s = eights(w)
    assert np.array_equal(unpacked(data.get(), rows, cols), q) and np.array_equal(scale.get(), s)
    q[0, :4] = -128
    dq, data = Dev(q), Dev(np.full(n, 0x55, np.uint8))
    to = R.RoasterI8(data.p, scale.p, rows, cols)
    R.check(R.lib().roaster_i8_pack(dq.p, R.I8_FROM_I8, C.byref(to)), "pack")
    sync()
    assert np.array_equal(unpacked(data.get(), rows, cols), q) and np.array_equal(scale.get(), s)
    assert np.array_equal(data.get().view(np.int8), packed(q).ravel())


def test_pack_rows_that_are_no_numbers():
    w = np.ones((3, 32), np.float32)
    w[0, 3], w[2, 31] = np.inf, np.nan
    dw, data, scale = Dev(w), Dev(np.zeros(R.lib().roaster_i8_bytes(3, 32), np.uint8)), Dev(np.zeros(3, np.float32))
    R.check(R.lib().roaster_i8_pack(dw.p, R.I8_FROM_F32, C.byref(R.RoasterI8(data.p, scale.p, 3, 32))), "pack")
    sync()
    v, s = unpacked(data.get(), 3, 32), scale.get()
    assert np.isnan(s[[0, 2]]).all() and not v[[0, 2]].any() and np.all(v[1] == 127) and s[1] == np.float32(1) / np.float32(127)


@pytest.mark.parametrize("q6", [0, 1])
def test_pack_quantised(q6):
    """Q4_K and Q6_K rows: the scale is the largest weight's, the values are within half a step of the weights (and the roundings of both)."""
    rows, cols = 37, 768
    raw = (R.synth_q6k if q6 else R.synth_q4k)(3, 9, rows * cols // 256)
    w = np.stack([O.matvec(q6, raw, np.eye(cols, dtype=np.float32)[c], rows, cols) for c in range(cols)], axis=1)
    dw, data, scale = Dev(raw), Dev(np.zeros(R.lib().roaster_i8_bytes(rows, cols), np.uint8)), Dev(np.zeros(rows, np.float32))
    to = R.RoasterI8(data.p, scale.p, rows, cols)
    R.check(R.lib().roaster_i8_pack(dw.p, R.I8_FROM_Q6K if q6 else R.I8_FROM_Q4K, C.byref(to)), "pack")
    sync()
    s = scale.get().astype(np.float64)
    top = np.abs(w).max(axis=1)
    assert np.all(np.abs(s - top / 127) <= 1e-5 * s)
    v = unpacked(data.get(), rows, cols)
    assert np.all(np.abs(v * s[:, None] - w) <= (0.5 + 127 * 1e-5) * s[:, None]) and np.all(np.abs(v).max(axis=1) == 127)
