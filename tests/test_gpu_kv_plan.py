"""roaster_kv_plan against a request-by-request plan on the host: equal in every
output, the table and the ring included."""
import numpy as np
import pytest

import roaster_amd as R
from attn_util import Plan, plan_oracle, pool, sync
from gpu_util import log

pytestmark = pytest.mark.gpu


def compare(p, want):
    got = p.got()
    for k, v in want.items():
        assert np.array_equal(got[k], v), (k, got[k], v)


def step(rng, n, page, hi, chunk, some=True):
    ln = rng.integers(0, hi + 1, n).astype(np.int32)
    kinds = rng.integers(0, 8, n)
    add = np.where(kinds == 0, -1, np.where(kinds == 1, 0, np.where(kinds == 2, chunk, 1))).astype(np.int32)
    return ln, add if some else np.ones(n, np.int32)


CASES = [(1, 16, 0, 1), (1, 4096, 9000, 5000), (3, 16, 40, 37), (8, 64, 6000, 1), (64, 32, 500, 100), (255, 16, 90, 20),
         (256, 16, 33, 3), (257, 128, 4000, 40), (700, 16, 3000, 11), (2048, 16, 50, 9), (2047, 256, 20000, 64)]


@pytest.mark.parametrize("n,page,hi,chunk", CASES)
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(n, page, hi, chunk, in_place):
    log(f"plan n={n} page={page} hi={hi} chunk={chunk} in_place={in_place}")
    rng = np.random.default_rng(n * 7 + page)
    ln, add = step(rng, n, page, hi, chunk)
    more = int(sum(-(-(l + max(a, 0)) // page) - -(-l // page) for l, a in zip(ln.tolist(), add.tolist())))
    width = -(-(hi + chunk) // page) + 1
    n_pages, table, ring, ctl = pool(rng, page, ln, more, width, front=5 * n + 11)
    rows = max(1, int(np.maximum(add, 0).sum()) + 13)
    want = plan_oracle(page, n_pages, rows, ln, add, table, ring, ctl)
    p = Plan(page, n_pages, rows, ln, add, table, ring, ctl, in_place)
    R.check(p.call(), "plan")
    sync()
    compare(p, want)
    if not in_place:                                   # the same call again: the same state
        R.check(p.call(), "plan")
        sync()
        compare(p, want)


@pytest.mark.parametrize("in_place", [False, True])
def test_many_rows(in_place):
    """Prompts of thousands of tokens: more workgroups than one, in place a second launch."""
    rng = np.random.default_rng(3)
    ln, add = np.array([0, 17, 70000, 3], np.int32), np.array([100000, -1, 9001, 120000], np.int32)
    n_pages, table, ring, ctl = pool(rng, 16, ln, 14400, 8000, front=3)
    want = plan_oracle(16, n_pages, 240000, ln, add, table, ring, ctl)
    p = Plan(16, n_pages, 240000, ln, add, table, ring, ctl, in_place)
    R.check(p.call(), "plan")
    sync()
    compare(p, want)


def test_steps_in_place_until_every_page_has_moved():
    """Requests that grow, end and start anew over many steps: pages go round the ring
    more than once, no page is held twice, and what is held and free stays whole."""
    rng = np.random.default_rng(9)
    n, page, width = 24, 16, 30
    n_pages, table, ring, ctl = pool(rng, page, np.zeros(n), 200, width, slack=0)
    ln = np.zeros(n, np.int32)
    for i in range(60):
        add = rng.integers(1, 40, n).astype(np.int32)
        add[(ln + add > 330) | (rng.random(n) < 0.15)] = -1
        need = -(-(ln + np.maximum(add, 0)) // page) - -(-ln // page)
        while need[add > 0].sum() > ctl[1] - ctl[0]:
            add[np.argmax(add)] = 0
        want = plan_oracle(page, n_pages, 1000, ln, add, table, ring, ctl)
        p = Plan(page, n_pages, 1000, ln, add, table, ring, ctl, in_place=i % 2 == 0)
        R.check(p.call(), "plan")
        sync()
        compare(p, want)
        got = p.got()
        ln, table, ring, ctl = got["len_out"], got["table"], got["ring"], got["ctl_out"]
        held = [table[r, j] for r in range(n) for j in range(-(-int(ln[r]) // page))]
        free = ring[np.arange(ctl[0], ctl[1]) % n_pages].tolist()
        assert sorted(held + free) == list(range(n_pages))
    assert ctl[1] > 2 * n_pages


def refused(rc, p, before, rows):
    R.check(p.call(), "plan")
    assert R.lib().roaster_sync() == rc, R.last_error()
    sync()                                             # reported once
    ln, table, ring, ctl = before
    compare(p, dict(len_out=ln, table=table, ring=ring, ctl_out=ctl, first=np.zeros(len(ln) + 1, np.int32),
                    row_req=np.full(rows, -1), row_pos=np.full(rows, -1), row_slot=np.full(rows, -1)))


@pytest.mark.parametrize("what", ["pages", "rows", "width", "negative", "long", "below", "ring", "front", "freed", "sum"])
@pytest.mark.parametrize("in_place", [False, True])
def test_step_refused_as_a_whole(what, in_place):
    rng = np.random.default_rng(5)
    ln, add = np.array([30, 64, 5, 100], np.int32), np.array([3, 10, -1, 1], np.int32)
    rows, width = 20, 8
    n_pages, table, ring, ctl = pool(rng, 16, ln, 1, width, slack=0)
    rc = R.EINVAL
    if what == "pages":                                # three are needed, one is free (the ended request's come behind)
        add[3], rows, rc = 13, 40, R.ENOMEM
    if what == "rows":
        rows = 13
    if what == "width":
        add[1] = 65
        rows = 200
    if what == "negative":
        ln[2] = -1
    if what == "long":
        ln[2] = 2 ** 31 - 1
    if what == "below":
        add[0] = -2
    if what == "ring":
        ctl[1] += n_pages
    if what == "front":
        ctl[0] = -1
    if what == "freed":                                # more pages come back than there can be
        ctl[1] += n_pages - (ctl[1] - ctl[0])
    if what == "sum":
        add[:] = 20
    p = Plan(16, n_pages, rows, ln, add, table, ring, ctl, in_place)
    refused(rc, p, (ln, table, ring, ctl), rows)


def test_bad_page_numbers_are_marked():
    """Pages out of range in the ring and in a table row: those rows get slot -1, others theirs."""
    ln, add = np.array([20, 16, 40], np.int32), np.array([1, 1, 1], np.int32)
    table = np.array([[4, 99, -1], [2, -1, -1], [5, 3, 1]], np.int32)
    ring = np.array([100, 6, 7, 8, 9, 0, 0, 0, 0, 0], np.int32)
    ctl = np.array([0, 3], np.int64)
    p = Plan(16, 10, 4, ln, add, table, ring, ctl)
    R.check(p.call(), "plan")
    assert R.lib().roaster_sync() == R.EINVAL
    sync()
    got = p.got()
    assert got["row_slot"].tolist() == [-1, -1, 16 + 8, -1] and got["row_req"].tolist() == [0, 1, 2, -1]
    assert got["table"].tolist() == [[4, 99, -1], [2, -1, -1], [5, 3, 1]] and got["ctl_out"].tolist() == [1, 3]


@pytest.mark.parametrize("in_place", [False, True])
def test_bad_pages_of_an_ended_request(in_place):
    """Page numbers out of range among those that come back: reported in this step and entered as
    -1, the others as they are; reported again in the step that takes one."""
    ln, add = np.array([50, 16], np.int32), np.array([-1, 0], np.int32)
    table = np.array([[4, 99, -7, 2, 55], [6, -1, -1, -1, -1]], np.int32)
    ring = np.array([0, 0, 0, 0, 0, 0, 0, 1, 8, 0], np.int32)
    ctl = np.array([7, 9], np.int64)
    p = Plan(16, 10, 4, ln, add, table, ring, ctl, in_place)
    R.check(p.call(), "plan")
    assert R.lib().roaster_sync() == R.EINVAL
    sync()
    got = p.got()
    assert got["ring"].tolist() == [-1, -1, 2, 0, 0, 0, 0, 1, 8, 4] and got["ctl_out"].tolist() == [7, 13]
    assert got["table"].tolist() == table.tolist() and got["len_out"].tolist() == [0, 16]
    p = Plan(16, 10, 64, got["len_out"], np.array([49, 0], np.int32), got["table"], got["ring"], got["ctl_out"], in_place)
    R.check(p.call(), "plan")
    assert R.lib().roaster_sync() == R.EINVAL
    sync()
    got = p.got()
    assert got["table"].tolist()[0] == [1, 8, 4, -1, 55] and got["ctl_out"].tolist() == [11, 13]
    assert got["row_slot"].tolist()[:49] == [pg * 16 + i for pg in (1, 8, 4) for i in range(16)] + [-1]
