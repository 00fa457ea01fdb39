"""roaster_matmul_i8: every kernel that it can choose, at sizes that fill none of its tiles.

KERNELS is the choice as the sizes make it; the cases are held to it, so that a change of the rule
shows which kernel has lost its tests.  Bounds as in test_gpu_i8.py."""
import ctypes as C

import numpy as np
import pytest

import roaster_amd as R
from attn_util import EPS24, sync
from gpu_util import Dev
from mixer_util import packed
from test_gpu_i8 import check, matmul, values
from test_gpu_mixer_offsets import FAR, Rows

pytestmark = pytest.mark.gpu


def kernel(T, N, K):
    """16 channels of up to 16 or 32 tokens and how many waves, or a tile's tokens / 32, channels / 128 and columns / 64 of a step."""
    up = lambda a, b: -(-a // b)  # noqa: E731
    if T <= 32 or up(T, 32) * up(N, 16) <= 256:
        return "few", 1 if T <= 16 else 2, 4 if K <= 8192 else 8
    if up(T, 128) * up(N, 256) >= 384:
        return "tile", 4, 2, 1
    return ("tile", 1, 1, 4) if up(T, 32) * up(N, 128) <= 256 else ("tile", 2, 1, 2)


TILES = [("tile", 4, 2, 1), ("tile", 1, 1, 4), ("tile", 2, 1, 2)]
KERNELS = [("few", t, w) for t in (1, 2) for w in (4, 8)] + TILES
# columns: one padded block, blocks that end inside a step of 256, an odd number of steps, and a long row
SIZES = [(T, N, K) for T, N in ((2047, 6401), (100, 2502), (300, 8197), (13, 37), (61, 515)) for K in (16, 272, 2064)] + \
    [(5, 35, 8208), (40, 70, 16384), (129, 4099, 8208), (3457, 3586, 144)]


def test_the_sizes_come_to_every_kernel():
    assert {kernel(*z) for z in SIZES} == set(KERNELS)
    for K in (16, 272, 2064):
        assert {kernel(*z) for z in SIZES if z[2] == K} >= set(TILES)


@pytest.mark.parametrize("T,N,K", SIZES)
def test_matmul(T, N, K):
    rng = np.random.default_rng(T + N + K)
    (xq, xs), (wq, ws) = values(rng, T, K), values(rng, N, K)
    check(matmul(xq, xs, wq, ws, x_pad=16 * (K % 3), y_pad=N % 4), xq, xs, wq, ws)


@pytest.mark.parametrize("T,N", [(70, 40), (70, 1700), (270, 4099), (3457, 3585)])
def test_largest_sums(T, N):
    """Every product at its largest over the longest rows: 2^30."""
    K = 65536
    assert kernel(T, N, K) == dict([(40, KERNELS[3]), (1700, TILES[1]), (4099, TILES[2]), (3585, TILES[0])])[N]
    xq, wq = np.full((T, K), -128, np.int8), np.full((N, K), -128, np.int8)
    wq[1::2] = 127
    got = matmul(xq, np.ones(T, np.float32), wq, np.ones(N, np.float32))
    assert np.all(got[:, ::2] == 2.0 ** 30) and np.all(got[:, 1::2] == -128 * 127 * 65536.0)


@pytest.mark.parametrize("T,N,want", [(150, 2500, TILES[1]), (150, 9000, TILES[2]), (1900, 7000, TILES[0])])
def test_odd_scales_stay_in_their_rows(T, N, want):
    assert kernel(T, N, 64) == want
    rng = np.random.default_rng(T)
    (xq, xs), (wq, ws) = values(rng, T, 64), values(rng, N, 64)
    xs[2], xs[T - 1], ws[11], ws[N - 1], ws[N // 2] = np.nan, np.inf, np.nan, 0, np.inf
    got = matmul(xq, xs, wq, ws)
    rows, cols = np.ones(T, bool), np.ones(N, bool)
    rows[[2, T - 1]], cols[[11, N // 2]] = False, False
    assert np.isnan(got[2]).all() and np.isnan(got[:, 11]).all() and not got[rows][:, N - 1].any()
    assert not np.isfinite(got[T - 1]).any() and not np.isfinite(got[:, N // 2]).any()
    check(got[rows][:, cols], xq[rows], xs[rows], wq[cols], ws[cols])


@pytest.mark.parametrize("N,want", [(2064, TILES[1]), (16500, TILES[2]), (98306, TILES[0])])
def test_rows_far_apart(N, want):
    """40 rows of both tensors 2^28 elements apart: most of them 4 GB and more behind the first."""
    T, K = 40, 160
    assert kernel(T, N, K) == want
    rng = np.random.default_rng(N)
    (xq, xs), (wq, ws) = values(rng, T, K), values(rng, N, K)
    dx, dy = Rows(T, K, np.int8).put(xq), Rows(T, N, np.float32)
    dw, dxs, dws = Dev(packed(wq)), Dev(xs), Dev(ws)
    try:
        a = R.RoasterMatmulI8(T, dx.p, FAR, dxs.p, dy.p, FAR)
        R.check(R.lib().roaster_matmul_i8(C.byref(a), C.byref(R.RoasterI8(dw.p, dws.p, N, K))), "matmul_i8")
        sync()
        want = (xq.astype(np.float64) @ wq.astype(np.float64).T) * xs[:, None].astype(np.float64) * ws.astype(np.float64)
        assert np.all(np.abs(dy.get() - want) <= 3 * EPS24 * 1.01 * np.abs(want))
    finally:
        dx.free()
        dy.free()
