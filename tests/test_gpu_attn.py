"""roaster_attn_paged against softmax attention in 64 bits, the error bound derived
in attn_util.attn_bound.  What a row must not use -- tokens behind its position,
pages of nobody, table entries past its last page -- holds NaN, infinities and
wild numbers throughout."""
import ctypes as C

import numpy as np
import pytest

import roaster_amd as R
from attn_util import Attn, Cache, attn_oracle, check_attn, sync
from gpu_util import Dev, log

pytestmark = pytest.mark.gpu


def make(rng, lens, KV, D, page, f16, spare=3):
    """A cache with `lens` tokens of each request in shuffled pages, poison elsewhere."""
    used = [-(-l // page) for l in lens]
    n_pages = sum(used) + spare
    ids = rng.permutation(n_pages).astype(np.int32)
    width = max(1, max(used)) + 2
    table = rng.choice(np.array([-5, 2 ** 30, n_pages, -2 ** 31], np.int32), (len(lens), width)).astype(np.int32)
    dt = np.float16 if f16 else np.float32
    kc, vc = (rng.choice(np.array([np.nan, np.inf, -np.inf], dt), (n_pages, KV, page, D)) for _ in range(2))
    at = 0
    for r, (l, u) in enumerate(zip(lens, used)):
        table[r, :u] = ids[at:at + u]
        for j in range(u):
            m = min(page, l - j * page)
            kc[ids[at + j], :, :m] = rng.standard_normal((KV, m, D)).astype(dt)
            vc[ids[at + j], :, :m] = (rng.standard_normal((KV, m, D)) + 0.2).astype(dt)
        at += u
    return kc, vc, table


def run_case(lens, rows, H, KV, D, page, f16, gate=False, peak=1.0, seed=0, scale=None):
    """rows: (request, position) of each row."""
    rng = np.random.default_rng(seed + 17 * len(lens) + D + page)
    kc, vc, table = make(rng, lens, KV, D, page, f16)
    rows = np.array(rows, np.int32).reshape(-1, 2)
    T = len(rows)
    q = (peak * rng.standard_normal((T, H, D))).astype(np.float32)
    g = rng.standard_normal((T, H, 2, D)).astype(np.float32) if gate else None
    scale = D ** -0.5 if scale is None else scale
    c = Cache(kc, vc)
    a = Attn(c, q, rows[:, 0].copy(), rows[:, 1].copy(), table, scale, g)
    R.check(a.call(), "attn")
    sync()
    got = a.out.get()
    want, mass, reach = attn_oracle(q, kc, vc, table, rows[:, 0], rows[:, 1], np.float64(np.float32(scale)),
                                    g[:, :, 1] if gate else None)
    skip = rows[:, 0] == -1
    assert np.all(got[skip] == 77)
    assert not got[(rows[:, 1] == -1) & ~skip].any()
    rel = check_attn(got[~skip], want[~skip], mass[~skip], reach[~skip], int(rows[:, 1].max()) + 1, D)
    # again on the same buffers: the same bits
    R.check(a.call(), "attn")
    sync()
    assert np.array_equal(a.out.get().view(np.uint32), got.view(np.uint32))
    return rel


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 127, 128, 129, 255, 256, 257, 500, 1025]
HEADS = [(16, 2, 256), (4, 4, 256), (32, 8, 128), (7, 1, 128), (20, 4, 64), (16, 1, 64), (24, 2, 128), (2, 1, 256)]


@pytest.mark.parametrize("H,KV,D", HEADS)
@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("page", [16, 64])
def test_one_row_a_request_of_every_length(H, KV, D, f16, page):
    log(f"attn H={H} KV={KV} D={D} f16={f16} page={page}")
    rel = run_case(EDGES, [(r, l - 1) for r, l in enumerate(EDGES)], H, KV, D, page, f16, gate=True)
    log(f"  rel {rel:.2e}")


@pytest.mark.parametrize("length", [1, 33, 300, 4097])
@pytest.mark.parametrize("f16", [True, False])
def test_one_request(length, f16):
    for H, KV, D in HEADS[:1] + HEADS[3:5]:
        log(f"attn one request length={length} H={H} KV={KV} D={D} f16={f16}")
        run_case([length], [(0, length - 1)], H, KV, D, 256, f16, gate=length == 300)


@pytest.mark.parametrize("page", [32, 4096])
def test_long_rows_next_to_short_ones(page):
    lens = [20000, 1, 0, 7, 3000, 40]
    run_case(lens, [(r, l - 1) for r, l in enumerate(lens)], 16, 2, 256, page, True, gate=True)


@pytest.mark.parametrize("f16", [True, False])
def test_peaked_softmax(f16):
    """Scores of +-60 and more: one position takes nearly all."""
    for H, KV, D in HEADS[:1] + HEADS[2:3]:
        run_case([700, 90], [(0, 699), (1, 89)], H, KV, D, 16, f16, peak=20.0)


def test_scales():
    for s in (0.0, -0.3, 1e-20, 1.0):
        run_case([200], [(0, 199)], 16, 2, 256, 16, True, scale=s)


CHUNKS = [
    ([300], [(0, p) for p in range(300)]),                                            # a prompt from its first token
    ([900], [(0, p) for p in range(644, 900)]),                                       # a chunk behind a context
    ([70, 200, 33], [(0, p) for p in range(60, 70)] + [(1, p) for p in range(100, 200)] + [(2, p) for p in range(33)]),
    ([40, 50], [(0, 39), (1, 49), (0, 38), (1, 3), (-1, -1), (0, 5), (0, 5), (1, -1), (0, 39)]),      # no order at all
    ([200], [(0, -1), (0, -1), (0, 100), (0, 150)] + [(0, -1)] + [(0, p) for p in range(120, 140)] + [(0, 7)]),
    ([120, 64], [(0, p) for p in range(100, 120)] + [(-1, -1)] * 5 + [(1, p) for p in range(60, 64)] + [(-1, -1)] * 40),
]


@pytest.mark.parametrize("i", range(len(CHUNKS)))
@pytest.mark.parametrize("H,KV,D", [HEADS[0], HEADS[2], HEADS[3], HEADS[4], HEADS[5]])
@pytest.mark.parametrize("f16", [True, False])
def test_several_rows_a_request(i, H, KV, D, f16):
    lens, rows = CHUNKS[i]
    log(f"attn chunk {i} H={H} KV={KV} D={D} f16={f16}")
    run_case(lens, rows, H, KV, D, 32, f16, gate=True)


@pytest.mark.parametrize("H,KV,D", HEADS)
@pytest.mark.parametrize("f16", [True, False])
def test_drafts_of_many_requests(H, KV, D, f16):
    """Two or three rows to a request, some skipped or without a position, of lengths that end
    within a tile and at its edge: 80 units at least."""
    rng = np.random.default_rng(H + D)
    lens = rng.integers(3, 200, 40).tolist() + [3, 16, 17, 18, 33, 3000]
    rows = []
    for r, l in enumerate(lens):
        n = 2 + r % 2
        rows += [(r, l - n + i) for i in range(n)]
        if r % 7 == 3:
            rows[-1] = (-1, 5)
        if r % 7 == 5:
            rows[-2] = (r, -1)
    run_case(lens, rows, H, KV, D, 16, f16, gate=True)


def test_many_rows_of_many_requests():
    """More rows than a launch has workgroups."""
    rng = np.random.default_rng(4)
    lens = rng.integers(1, 40, 700).tolist()
    run_case(lens, [(r, l - 1) for r, l in enumerate(lens)], 4, 2, 64, 16, True)


def test_pages_shared_by_requests():
    """Two requests with the same first pages, as a shared prompt has."""
    rng = np.random.default_rng(8)
    kc, vc, table = make(rng, [64, 20], 2, 128, 16, True)
    table = np.stack([table[0], table[0]])
    table[1, 3] = table[0, 0]
    q = rng.standard_normal((2, 8, 128)).astype(np.float32)
    req, pos = np.array([0, 1], np.int32), np.array([63, 55], np.int32)
    a = Attn(Cache(kc, vc), q, req, pos, table, 0.1)
    R.check(a.call(), "attn")
    sync()
    check_attn(a.out.get(), *attn_oracle(q, kc, vc, table, req, pos, np.float64(np.float32(0.1))), 64, 128)


def test_infinite_and_nan_values_in_use():
    """An infinite value reaches the heads that weigh it and no others' dims; a NaN key makes its rows NaN."""
    rng = np.random.default_rng(2)
    for f16 in (True, False):
        kc, vc, table = make(rng, [50, 50], 2, 128, 16, f16)
        vc[table[0, 3], 0, 1, 5] = np.inf              # the last token, in a tile's tail
        kc[table[1, 0], 1, 2, 7] = np.nan
        q = rng.standard_normal((2, 4, 128)).astype(np.float32)
        req, pos = np.array([0, 1], np.int32), np.array([49, 49], np.int32)
        a = Attn(Cache(kc, vc), q, req, pos, table, 0.1)
        R.check(a.call(), "attn")
        sync()
        got = a.out.get()
        assert np.all(np.isposinf(got[0, :2, 5])) and np.all(np.isnan(got[1, 2:]))
        assert np.isfinite(np.delete(got[0, :2], 5, axis=1)).all() and np.isfinite(got[0, 2:]).all()
        assert np.isfinite(got[1, :2]).all()


@pytest.mark.parametrize("size", [1e-12, 1e-3, 1e4, 1e15])
def test_queries_of_any_size(size):
    """Queries far from 1, the scale making up for it: the fp16 parts go by the row's own size."""
    rng = np.random.default_rng(6)
    kc, vc, table = make(rng, [130], 2, 256, 16, True)
    q = (size * rng.standard_normal((1, 16, 256))).astype(np.float32)
    q[0, 3] = 0
    req, pos = np.zeros(1, np.int32), np.array([129], np.int32)
    scale = np.float32(1 / (16 * size))
    a = Attn(Cache(kc, vc), q, req, pos, table, float(scale))
    R.check(a.call(), "attn")
    sync()
    check_attn(a.out.get(), *attn_oracle(q, kc, vc, table, req, pos, np.float64(scale)), 130, 256)


def test_rows_behind_the_count_stay():
    rng = np.random.default_rng(3)
    kc, vc, table = make(rng, [40], 2, 64, 16, True)
    q = rng.standard_normal((5, 4, 64)).astype(np.float32)
    req, pos = np.zeros(5, np.int32), np.full(5, 39, np.int32)
    a = Attn(Cache(kc, vc), q, req, pos, table, 0.125, rows=3)
    R.check(a.call(), "attn")
    sync()
    got = a.out.get()
    assert np.all(got[3:] == 77) and not np.any(got[:3] == 77)


@pytest.mark.parametrize("f16", [True, False])
def test_bad_rows_are_nan_and_reported(f16):
    """Requests, positions and pages out of range: NaN in those rows, the others right."""
    rng = np.random.default_rng(7)
    lens = [50, 60, 40, 3000]
    kc, vc, table = make(rng, lens, 2, 128, 16, f16)
    n_pages, width = kc.shape[0], table.shape[1]
    bad = table.copy()
    bad[1, 2], bad[2, 0] = n_pages, -1
    rows = [(0, 49), (1, 59), (1, 31), (2, 39), (4, 3), (-2, 3), (0, -2), (0, 16 * width), (3, 2999), (0, 2 ** 31 - 1),
            (0, -2 ** 31)] + [(0, 20)] * 30
    rows = np.array(rows, np.int32)
    q = rng.standard_normal((len(rows), 8, 128)).astype(np.float32)
    a = Attn(Cache(kc, vc), q, rows[:, 0].copy(), rows[:, 1].copy(), bad, 0.1)
    R.check(a.call(), "attn")
    assert R.lib().roaster_sync() == R.EINVAL
    sync()
    got = a.out.get()
    good = np.array([i for i in range(len(rows)) if i in (0, 2, 8) or i > 10])
    assert all(np.isnan(got[i]).all() for i in range(len(rows)) if i not in good)
    want = attn_oracle(q[good], kc, vc, table, rows[good, 0], rows[good, 1], np.float64(np.float32(0.1)))
    check_attn(got[good], *want, 3000, 128)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("T,at", [(3, 60), (24, 60), (24, 3000), (4, 3000)])
def test_a_bad_page_is_of_the_rows_that_reach_it(f16, T, at):
    """Rows of one request before and behind a bad page, together in one call: the
    former are right, the latter NaN."""
    rng = np.random.default_rng(T + at)
    kc, vc, table = make(rng, [at + T], 2, 128, 16, f16)
    bad = table.copy()
    split = (at + T // 2) // 16 * 16                   # the bad page's first token
    bad[0, split // 16] = kc.shape[0]
    pos = np.array([split - 1 - T // 2 + i for i in range(T)], np.int32)
    req = np.zeros(T, np.int32)
    q = rng.standard_normal((T, 8, 128)).astype(np.float32)
    a = Attn(Cache(kc, vc), q, req, pos, bad, 0.1)
    R.check(a.call(), "attn")
    assert R.lib().roaster_sync() == R.EINVAL
    sync()
    got = a.out.get()
    good = np.flatnonzero(pos < split)
    assert 0 < len(good) < T and np.isnan(got[len(good):]).all()
    want = attn_oracle(q[good], kc, vc, table, req[good], pos[good], np.float64(np.float32(0.1)))
    check_attn(got[good], *want, int(pos[-1]) + 1, 128)


@pytest.mark.parametrize("H,KV,D,lens,each", [
    (2, 1, 64, [730], 700),                            # more rows than a workgroup has threads, few columns
    (32, 8, 128, [600], 512),                          # 128 units in equal parts
    (4, 4, 64, [900, 40, 17, 300, 2000], 40),          # unequal requests
    (16, 2, 64, [5000] + [24] * 30, 24),               # one long request among short ones: equal parts would be too long
])
def test_chunks_of_every_split(H, KV, D, lens, each):
    rows = [(r, max(l - each, 0) + i) for r, l in enumerate(lens) for i in range(min(each, l))]
    run_case(lens, rows, H, KV, D, 32, True, gate=True)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("H,KV,D", [(16, 2, 256), (32, 8, 128), (4, 4, 64)])
@pytest.mark.parametrize("n,each", [(1, 3), (1, 40), (40, 2), (40, 3), (20, 5)])
def test_odd_values_reach_only_the_rows_that_use_them(n, each, H, KV, D, f16):
    """Infinite and NaN values at positions of a call's own rows: the rows before them are
    right, in those from there on the elements of these values are infinite or NaN, the others right."""
    rng = np.random.default_rng(n + each + D)
    lens = [int(l) for l in rng.integers(each, 260, n)]
    kc, vc, table = make(rng, lens, KV, D, 16, f16)
    rows = np.array([(r, l - each + i) for r, l in enumerate(lens) for i in range(each)], np.int32)
    for r, l in enumerate(lens):
        if r % 4 != 3:
            at = l - each + 1 + int(rng.integers(0, each - 1))
            for e in rng.integers(0, D, 4):
                vc[table[r, at // 16], :, at % 16, e] = [np.nan, np.inf, -np.inf][int(e) % 3]
    q = rng.standard_normal((len(rows), H, D)).astype(np.float32)
    a = Attn(Cache(kc, vc), q, rows[:, 0].copy(), rows[:, 1].copy(), table, D ** -0.5)
    R.check(a.call(), "attn")
    sync()
    got = a.out.get()
    with np.errstate(invalid="ignore"):
        want, mass, reach = attn_oracle(q, kc, vc, table, rows[:, 0], rows[:, 1], np.float64(np.float32(D ** -0.5)))
    fin = np.isfinite(want)
    assert not fin.all() and fin[::each].all()
    assert np.array_equal(np.isfinite(got), fin)
    check_attn(np.where(fin, got, 0), np.where(fin, want, 0), np.where(fin, mass, 0), reach, 260, D)


def test_cache_past_32_bit_offsets():
    """Pages beyond 2^32 elements of a cache of 9 GB for the keys and as much for the values."""
    L = R.lib()
    KV, D, page, n_pages = 2, 256, 64, 140000
    size = KV * page * D * 2
    rng = np.random.default_rng(12)
    lens = [64 * 5 + 9]
    kc, vc, table = make(rng, lens, KV, D, page, True, spare=0)
    ids = np.array([n_pages - 1 - 2 * i for i in range(6)], np.int32)
    assert (int(ids.min()) * size) // 2 > 2 ** 32
    k, v = (L.roaster_dev_alloc(n_pages * size) for _ in range(2))
    assert k and v, R.last_error()
    try:
        for i in range(6):
            for base, c in ((k, kc), (v, vc)):
                part = np.ascontiguousarray(c[table[0, i]])
                R.check(L.roaster_h2d(base + int(ids[i]) * size, part.ctypes.data, size), "h2d")
        far = table.copy()
        far[0, :6] = ids
        q = rng.standard_normal((1, 16, D)).astype(np.float32)
        req, pos = np.zeros(1, np.int32), np.array([lens[0] - 1], np.int32)
        c = Cache(kc, vc)
        a = Attn(c, q, req, pos, far, 0.0625)
        c.c.k, c.c.v, c.c.n_pages = k, v, n_pages
        R.check(a.call(), "attn")
        sync()
        check_attn(a.out.get(), *attn_oracle(q, kc, vc, table, req, pos, 0.0625), lens[0], D)
    finally:
        L.roaster_dev_free(k)
        L.roaster_dev_free(v)


@pytest.mark.parametrize("size", [1e-30, 1e34, 3e38])
@pytest.mark.parametrize("H,KV,D", [(16, 2, 256), (32, 8, 128), (7, 1, 64)])
def test_f32_values_of_any_size(H, KV, D, size):
    """Outputs are means of values, within f32 where the values are."""
    rng = np.random.default_rng(D)
    for lens, each in (([300], 1), ([70, 3, 41], 1), ([60 + i for i in range(40)], 2), ([80], 30)):
        kc, vc, table = make(rng, lens, KV, D, 16, False)
        vc = np.where(np.isfinite(vc), np.float32(size) * rng.uniform(-1, 1, vc.shape), vc).astype(np.float32)
        rows = np.array([(r, l - each + i) for r, l in enumerate(lens) for i in range(each)], np.int32)
        q = rng.standard_normal((len(rows), H, D)).astype(np.float32)
        a = Attn(Cache(kc, vc), q, rows[:, 0].copy(), rows[:, 1].copy(), table, D ** -0.5)
        R.check(a.call(), "attn")
        sync()
        want, mass, reach = attn_oracle(q, kc, vc, table, rows[:, 0], rows[:, 1], np.float64(np.float32(D ** -0.5)))
        check_attn(a.out.get() / size, want / size, mass / size, reach, int(rows[:, 1].max()) + 1, D)


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("H,KV,D", [(16, 2, 256), (16, 1, 64), (8, 2, 128)])
def test_rows_without_a_position_are_zero_whatever_their_gate(H, KV, D, f16):
    """Alone, among requests' rows, at the beginning of a run, and where a run's parts are joined."""
    rng = np.random.default_rng(D + H)
    for lens, rows in (([50], [(0, -1)]), ([50, 9], [(0, 49), (1, -1), (0, -1)]),
                       ([40 + i for i in range(60)], [(r, -1 if r % 3 else 39 + r) for r in range(60)]),
                       ([40 + i for i in range(40)], [(r, p) for r in range(40) for p in (-1, 39 + r)]),
                       ([3000], [(0, -1)] * 5 + [(0, 2970 + i) for i in range(25)])):
        kc, vc, table = make(rng, lens, KV, D, 16, f16)
        rows = np.array(rows, np.int32)
        q = rng.standard_normal((len(rows), H, D)).astype(np.float32)
        none = rows[:, 1] == -1
        g = rng.standard_normal((len(rows), H, 2, D)).astype(np.float32)
        g[none, :, 1] = rng.choice(np.array([np.nan, np.inf, -np.inf, 1], np.float32), (int(none.sum()), H, D))
        a = Attn(Cache(kc, vc), q, rows[:, 0].copy(), rows[:, 1].copy(), table, D ** -0.5, g)
        R.check(a.call(), "attn")
        sync()
        got = a.out.get()
        assert not got[none].any(), np.isnan(got[none]).sum()
        if not none.all():
            want = attn_oracle(q, kc, vc, table, rows[:, 0], rows[:, 1], np.float64(np.float32(D ** -0.5)),
                               np.where(np.isfinite(g[:, :, 1]), g[:, :, 1], 0))
            check_attn(got[~none], *(w[~none] for w in want), int(rows[:, 1].max()) + 1, D)
