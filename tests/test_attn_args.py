"""What the attention operators refuse (include/roaster_attn.h), on the CPU: every
argument check runs before the device is touched, so a refused call returns
ROASTER_EINVAL here too and an accepted one comes as far as the missing GPU.
And the index functions the kernels use (attn_index.h), over good and bad
values of everything that only the device sees."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

import roaster_amd as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "roaster_amd", "csrc")
BASE = 1 << 40                                        # addresses that are only looked at


def mem(i):
    return BASE + (i << 34)


def cache(**kw):
    d = dict(k=mem(1), v=mem(2), type=R.KV_F16, n_pages=100, page_size=64, kv_heads=2, head_dim=256)
    d.update(kw)
    return R.RoasterKvCache(**d)


def plan(**kw):
    d = dict(n_req=8, page_size=64, n_pages=100, max_pages=20, max_rows=16, len=mem(3), add=mem(4), len_out=mem(5),
             table=mem(6), ring=mem(7), ctl=mem(8), ctl_out=mem(9), first=mem(10), row_req=mem(11), row_pos=mem(12),
             row_slot=mem(13))
    d.update(kw)
    return R.lib().roaster_kv_plan(C.byref(R.RoasterKvPlan(**d)))


def rope(c=None, **kw):
    d = dict(rows=5, q_heads=16, q=mem(3), q_row=8192, q_head=512, k=mem(4), k_row=512, k_head=256, v=mem(5), v_row=512,
             v_head=256, q_norm=mem(6), k_norm=mem(7), eps=1e-6, rot_dim=64, pair_adjacent=0, theta=1e7, row_pos=mem(8),
             row_slot=mem(9), q_out=mem(10))
    d.update(kw)
    return R.lib().roaster_qk_rope_store(C.byref(R.RoasterQkRope(**d)), C.byref(c or cache()))


def attn(c=None, **kw):
    c = c or cache()
    d = dict(rows=5, q_heads=16, q=mem(3), row_req=mem(4), row_pos=mem(5), table=mem(6), n_req=8, max_pages=20,
             scale=0.0625, gate=mem(7), gate_row=8192, gate_head=512, out=mem(8), ws=mem(9), ws_bytes=1 << 33)
    d.update(kw)
    return R.lib().roaster_attn_paged(C.byref(R.RoasterAttnPaged(**d)), C.byref(c))


no_gpu = pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="these addresses must not reach a GPU")


@no_gpu
def test_good_arguments_come_as_far_as_the_device():
    for call in (plan, rope, attn):
        assert call() == R.EDEVICE, (call, R.last_error())
    assert plan(first=None) == R.EDEVICE
    assert plan(len_out=mem(3), ctl_out=mem(8)) == R.EDEVICE          # in place
    assert rope(q_norm=None, k_norm=None, rot_dim=0) == R.EDEVICE
    assert rope(q_head=256, q_row=4096, q_out=mem(3)) == R.EDEVICE    # in place
    assert attn(gate=None, gate_row=3, gate_head=1) == R.EDEVICE      # strides of no gate
    assert rope(rows=0) == R.OK and attn(rows=0) == R.OK              # nothing to do


@pytest.mark.parametrize("kw", [
    dict(n_req=0), dict(n_req=2049), dict(max_rows=0), dict(max_rows=(1 << 18) + 1), dict(page_size=8), dict(page_size=48),
    dict(page_size=8192), dict(n_pages=0), dict(n_pages=1 << 25), dict(max_pages=0), dict(max_pages=(1 << 24) + 1),
    dict(len=None), dict(add=None), dict(len_out=None), dict(table=None), dict(ring=None), dict(ctl=None),
    dict(ctl_out=None), dict(row_req=None), dict(row_pos=None), dict(row_slot=None), dict(len=mem(3) + 2),
    dict(ctl=mem(8) + 4), dict(len_out=mem(3) + 4), dict(ctl_out=mem(8) + 8), dict(table=mem(7)), dict(first=mem(4) + 28),
    dict(row_slot=mem(11)), dict(ring=mem(3) - 396)])
def test_plan_refuses(kw):
    assert plan(**kw) == R.EINVAL, kw


BAD_CACHE = [dict(k=None), dict(v=None), dict(k=mem(1) + 8), dict(type=2), dict(type=-1), dict(n_pages=0), dict(page_size=8),
             dict(page_size=65), dict(page_size=8192), dict(n_pages=1 << 26), dict(kv_heads=0), dict(kv_heads=1025),
             dict(head_dim=96), dict(head_dim=512), dict(head_dim=0)]


@pytest.mark.parametrize("kw", BAD_CACHE)
def test_cache_refused(kw):
    c = cache(**kw)
    assert rope(c) == R.EINVAL and attn(c) == R.EINVAL
    assert R.lib().roaster_attn_ws_bytes(1, 16, C.byref(c)) == 0


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=(1 << 20) + 1), dict(q_heads=0), dict(q_heads=1025), dict(rot_dim=-8), dict(rot_dim=12),
    dict(rot_dim=264), dict(theta=0.0), dict(theta=-1.0), dict(theta=0.5), dict(theta=float("nan")), dict(theta=float("inf")), dict(q=None),
    dict(k=None), dict(v=None), dict(q_out=None), dict(q=mem(3) + 4), dict(v=mem(5) + 8), dict(q_out=mem(10) + 4),
    dict(q_row=4098), dict(k_head=255), dict(v_row=1 << 40), dict(row_pos=None), dict(row_slot=None),
    dict(row_pos=mem(8) + 1), dict(q_norm=mem(6) + 4), dict(q_out=mem(3)), dict(q_out=mem(3) + 4096), dict(q_out=mem(4)),
    dict(q_out=mem(1)), dict(v=mem(2) + 4096), dict(k_norm=mem(1)), dict(row_slot=mem(10))])
def test_rope_refuses(kw):
    assert rope(**kw) == R.EINVAL, kw


def test_rope_refuses_keys_over_values():
    assert rope(cache(v=mem(1) + 4096)) == R.EINVAL


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=(1 << 20) + 1), dict(q_heads=0), dict(q_heads=17), dict(q_heads=1026), dict(n_req=0),
    dict(max_pages=0), dict(max_pages=(1 << 24) + 1), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None),
    dict(row_req=None), dict(row_pos=None), dict(table=None), dict(out=None), dict(q=mem(3) + 8), dict(out=mem(8) + 4),
    dict(table=mem(6) + 2), dict(gate=mem(7) + 4), dict(gate_row=8190), dict(gate_head=510), dict(gate_row=1 << 40),
    dict(ws=None), dict(ws=mem(9) + 8), dict(ws_bytes=0), dict(out=mem(3)), dict(out=mem(1)), dict(ws=mem(2)),
    dict(out=mem(6)), dict(ws=mem(8) + 16)])
def test_attn_refuses(kw):
    assert attn(**kw) == R.EINVAL, kw


def test_workspace_is_checked_and_grows_with_nothing_but_the_call():
    c = cache()
    ws = lambda *a: R.lib().roaster_attn_ws_bytes(*a, C.byref(c))  # noqa: E731
    assert ws(0, 16) > 0 and ws(1 << 20, 1024) >= ws(1, 16) > 0
    assert ws(-1, 16) == 0 and ws(1, 15) == 0 and ws((1 << 20) + 1, 16) == 0 and ws(1, 0) == 0
    assert attn(c, ws_bytes=ws(5, 16) - 1) == R.EINVAL


PROGRAM = r"""
#include <limits.h>
#include <stdio.h>
#include "attn_index.h"
int main()
{
    const int odd[] = { INT_MIN, INT_MIN + 1, -64, -2, -1, 0, 1, 2, 63, 64, 65, 4095, 4096, INT_MAX - 1, INT_MAX };
    for (int shift = 4; shift <= 12; shift++)
        for (int n = 1; n <= 1 << 20; n *= 7)
            for (int kv = 1; kv <= 8; kv *= 8) {
                if (((long long)n << shift) > INT_MAX) continue;
                const KvShape s = { shift, n, kv, 256 };
                for (int p : odd)
                    for (int d = -1; d <= 1; d++) {
                        const int page = (p == INT_MIN && d < 0) || (p == INT_MAX && d > 0) ? p : p + d;
                        if (!s.page_ok(page)) { if (page >= 0 && page < n) return puts("page refused"), 1; continue; }
                        if (page < 0 || page >= n) return puts("page"), 1;
                        for (int h = 0; h < kv; h += kv > 1 ? kv - 1 : 1)
                            if (s.at(page, h, (1 << shift) - 1) + s.dim > s.elements()) return puts("element"), 1;
                    }
                for (int v : odd) {
                    const bool in = v >= 0 && v < (n << shift);
                    if (s.slot_ok(v) != in) return printf("slot %d of %d\n", v, n << shift), 1;
                    if (in && s.at_slot(v, kv - 1) + s.dim > s.elements()) return puts("slot element"), 1;
                }
                const KvTable t = { 5, n };
                for (int r : odd)
                    for (int p : odd) {
                        const int k = t.tokens(r, p, shift);
                        const bool in = r >= 0 && r < 5 && p >= -1 && p < ((long long)n << shift);
                        if ((k >= 0) != in) return printf("row %d %d\n", r, p), 1;
                        if (in && k != p + 1) return puts("tokens"), 1;
                        for (long long j = k - 1; j >= 0 && j >= k - 2; j--)
                            if (t.entry(r, (int)j, shift) >= (size_t)5 * n) return puts("entry"), 1;
                    }
            }
    return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_index_functions_stay_inside(tmp_path):
    src, exe = tmp_path / "index.cpp", tmp_path / "index"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-I", CSRC, "-o", str(exe), str(src)])
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and not r.stderr, r.stdout + r.stderr


@pytest.mark.parametrize("scale", [3e38, -3e38, 2.4e38, float("-inf")])
def test_scales_whose_product_with_log2_e_overflows_are_refused(scale):
    assert attn(scale=scale) == R.EINVAL


@no_gpu
def test_scales_up_to_that_are_taken():
    for scale in (2e38, -2e38, 0.0, 1e-38):
        assert attn(scale=scale) == R.EDEVICE
