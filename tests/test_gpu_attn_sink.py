"""roaster_attn_paged where one position outweighs the rest and its value is zero: the
output is what the other positions give, 2^-12 .. 2^-22 of the largest probability each.

Queries, keys and the scale are chosen so that a score, in octaves, is exact in the
kernels: elements are multiples of 1/8, eight of them count, and the f32 product of
scale and log2 e is 1.  What is left of an output's error, relative to
mass = sum_j p_j |v_j|:
  2 reach 2^-24       scale is ln 2 to half a step of f32
  2^-21               exp2 off by a step (2^-23) in a term and in the sum of the terms, and
                      2^-22 for a term's two fp16 parts ...
  2^-24 T / mass      ... or 2^-24 of the tile's largest term, the sink apart: T = (largest
                      term of the others) sum |v|
  32 2^-38 |v| / mass ... or 2^-38 of the sink where they share its tile of up to 32 tokens
  2 (n/16 + 48) 2^-23 the sums of values and of terms: a wave's tiles in turn, a tile's 16 or
                      32 products, the waves' and parts' joins
As a whole (norms) errors of many roundings are far smaller than their sum: 1e-5."""
import numpy as np
import pytest

import roaster_amd as R
from attn_util import EPS24, Attn, Cache, attn_oracle, sync
from gpu_util import log

pytestmark = pytest.mark.gpu
LN2 = np.float32(np.log(2))


def sink_case(lens, rows, H, KV, D, r, at, flat, f16=True, page=16):
    """Requests with one heavy position each, r octaves above the others' typical score, at
    token `at` (from the end if negative); `flat`: the others' scores are equal."""
    rng = np.random.default_rng(len(lens) + len(rows) + D + r)
    dt = np.float16 if f16 else np.float32
    used = [-(-l // page) for l in lens]
    ids = rng.permutation(sum(used)).astype(np.int32)
    table = np.full((len(lens), max(used)), -1, np.int32)
    kc, vc = (np.full((sum(used), KV, page, D), np.nan, dt) for _ in range(2))
    base = np.zeros(D)
    base[1:9] = [0.5, -0.25, 0.125, -0.5, 0.25, 0.375, -0.125, -0.25]
    first = 0
    for i, l in enumerate(lens):
        table[i, :used[i]] = ids[first:first + used[i]]
        first += used[i]
        k = np.round(8 * rng.standard_normal((l, KV, D))) / 8
        k[:, :, 1:9] = np.tile(np.abs(base[1:9]), (l, KV, 1)) if flat else k[:, :, 1:9]
        k[:, :, 0] = 0
        v = rng.uniform(0.5, 1.5, (l, KV, D)) if flat else rng.standard_normal((l, KV, D))
        s = at % l
        k[s], v[s] = 0, 0
        k[s, :, 0] = 16
        pg = table[i, np.arange(l) // page]
        kc[pg, :, np.arange(l) % page] = k
        vc[pg, :, np.arange(l) % page] = v
    rows = np.array(rows, np.int32)
    q = np.tile(base, (len(rows), H, 1)) * rng.choice([-1.0, 1.0], (len(rows), H, 1))
    q[:, :, 0] = r / 16
    q = q.astype(np.float32)
    assert LN2 * np.float32(1.44269504088896341) == 1
    a = Attn(Cache(kc, vc), q, rows[:, 0].copy(), rows[:, 1].copy(), table, float(LN2))
    R.check(a.call(), "attn")
    sync()
    got = a.out.get()
    want, mass, reach = attn_oracle(q, kc, vc, table, rows[:, 0], rows[:, 1], np.float64(LN2))
    lim = np.zeros_like(want)
    for t, (i, p) in enumerate(rows):
        n = int(p) + 1
        pg, o = table[i, np.arange(n) // page], np.arange(n) % page
        k, v = (c[pg, :, o].astype(np.float64) for c in (kc, vc))            # [n, KV, D]
        for h in range(H):
            s = k[:, h // (H // KV)] @ q[t, h].astype(np.float64)
            w = np.exp2(s - s.max())
            w /= w.sum()
            rest = np.where(k[:, 0, 0] == 16, 0, w)
            av = np.abs(v[:, h // (H // KV)])
            lim[t, h] = (mass[t, h] * (2 * reach[t, h] * EPS24 + 2.0 ** -21 + (n / 16 + 48) * 2.0 ** -22)
                         + 2.0 ** -24 * rest.max() * av.sum(0) + 32 * 2.0 ** -38 * av.max(0) + 1e-30)
    err = np.abs(got - want)
    worst, rel = float((err / lim).max()), float(np.linalg.norm(got - want) / np.linalg.norm(want))
    log(f"sink r={r} at={at} flat={flat} H={H} KV={KV} D={D} rows={len(rows)} f16={f16}: worst {worst:.3f} rel {rel:.2e}")
    assert worst <= 1
    assert rel <= 1e-5


FORMS = {
    "one": ([700], [(0, 699)]),
    "long": ([4097], [(0, 4096)]),
    "short": ([30, 500, 65], [(0, 29), (1, 499), (2, 64)]),
    "many": ([90 + 9 * i for i in range(70)], [(i, 89 + 9 * i) for i in range(70)]),
    "drafts": ([90 + 9 * i for i in range(40)], [(i, 87 + 9 * i + j) for i in range(40) for j in range(3)]),
    "rows": ([620], [(0, p) for p in range(600, 620)]),
    "chunk": ([700], [(0, p) for p in range(390, 700)]),
}


@pytest.mark.parametrize("r", [12, 17, 22])
@pytest.mark.parametrize("form", sorted(FORMS))
@pytest.mark.parametrize("H,KV,D", [(16, 2, 256), (16, 1, 64), (8, 2, 128)])
def test_a_heavy_position_without_a_value(form, H, KV, D, r):
    lens, rows = FORMS[form]
    for at, flat in ((0, True), (0, False), (37, True), (-1, False)):
        if at == -1 and len(rows) > len(lens):
            continue                                   # some of a request's rows would not reach it
        sink_case(lens, rows, H, KV, D, r, at, flat)


@pytest.mark.parametrize("form", ["one", "drafts", "rows"])
def test_the_same_in_an_f32_cache(form):
    lens, rows = FORMS[form]
    sink_case(lens, rows, 16, 2, 128, 22, 0, True, f16=False)


@pytest.mark.parametrize("form", ["long", "drafts", "chunk"])
def test_heavy_positions_on_the_way(form):
    """Scores that rise and fall over the whole length, 60 octaves between them: the sums'
    scale has to follow them up, and down, without overflow."""
    rng = np.random.default_rng(5)
    lens, rows = FORMS[form]
    H, KV, D, page = 16, 2, 128, 16
    used = [-(-l // page) for l in lens]
    table = np.full((len(lens), max(used)), -1, np.int32)
    kc = np.zeros((sum(used), KV, page, D), np.float16)
    vc = rng.standard_normal(kc.shape).astype(np.float16)
    first = 0
    for i, u in enumerate(used):
        table[i, :u] = np.arange(first, first + u)
        first += u
        x = np.arange(u * page)
        wave = np.round(8 * 30 * np.sin(x / (5 + 40 * rng.random())) * np.minimum(1, x / 200)) / 8
        kc[table[i, :u], :, :, 0] = wave.reshape(u, 1, page)
    rows = np.array(rows, np.int32)
    q = np.zeros((len(rows), H, D), np.float32)
    q[:, :, 0] = rng.choice([-1.0, 1.0, 0.5], (len(rows), H))
    a = Attn(Cache(kc, vc), q, rows[:, 0].copy(), rows[:, 1].copy(), table, float(LN2))
    R.check(a.call(), "attn")
    sync()
    got = a.out.get()
    want, mass, reach = attn_oracle(q, kc, vc, table, rows[:, 0], rows[:, 1], np.float64(LN2))
    n = int(rows[:, 1].max()) + 1
    # as above; a tile's largest term has a value of its own, so 2^-24 of it is 2^-24 / its |v| of its mass: to the norm
    rel = float(np.linalg.norm(got - want) / np.linalg.norm(want))
    log(f"waves {form}: rel {rel:.2e}")
    assert np.isfinite(got).all() and rel <= 1e-5
    lim = mass * (2 * reach[..., None] * EPS24 + 2.0 ** -21 + (n / 16 + 48) * 2.0 ** -22) + 2.0 ** -24 * np.abs(vc).max() * 32
    assert np.all(np.abs(got - want) <= lim)
