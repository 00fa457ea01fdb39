"""What the operators of a recurrent layer refuse (include/roaster_mixer.h), on the
CPU: every argument check runs before the device is touched, so a refused call
returns ROASTER_EINVAL here too and an accepted one comes as far as the missing GPU."""
import ctypes as C
import os

import pytest

import roaster_amd as R

BASE = 1 << 40                                        # addresses that are only looked at


def mem(i):
    return BASE + (i << 36)


def norm(**kw):
    d = dict(rows=5, cols=2048, group=2048, x=mem(1), x_row=2048, res=mem(2), res_row=2048, weight=mem(3), gate=mem(4), gate_row=4096,
             eps=1e-6, y=mem(5), y_row=2048, q=mem(6), q_row=2048, q_scale=mem(7))
    d.update(kw)
    return R.lib().roaster_norm(C.byref(R.RoasterNorm(**d)))


def i8(**kw):
    d = dict(data=mem(1), scale=mem(2), rows=100, cols=512)
    d.update(kw)
    return R.RoasterI8(**d)


def pack(W=mem(3), kind=R.I8_FROM_F32, **kw):
    return R.lib().roaster_i8_pack(W, kind, C.byref(i8(**kw)))


def matmul(w=None, **kw):
    d = dict(rows=7, x=mem(3), x_row=512, x_scale=mem(4), y=mem(5), y_row=100)
    d.update(kw)
    return R.lib().roaster_matmul_i8(C.byref(R.RoasterMatmulI8(**d)), C.byref(w or i8()))


def state(**kw):
    d = dict(n_req=8, k_heads=16, v_heads=32, k_dim=128, v_dim=128, taps=4, conv=mem(1), state=mem(2))
    d.update(kw)
    return R.RoasterSsmState(**d)


def scan(s=None, **kw):
    d = dict(rows=64, most=20, mode=R.SCAN_DELTA, x=mem(3), x_row=8192, a=mem(4), a_row=32, b=mem(5), b_row=32, conv_w=mem(6),
             conv_b=mem(7), a_coef=mem(8), dt_bias=mem(9), skip=mem(10), scale=0.1, eps=1e-6, first=mem(11), row_pos=mem(12),
             out=mem(13), out_row=4096, ws=mem(14), ws_bytes=1 << 35)
    d.update(kw)
    return R.lib().roaster_ssm_scan(C.byref(R.RoasterSsmScan(**d)), C.byref(s or state()))


no_gpu = pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="these addresses must not reach a GPU")


@no_gpu
def test_good_arguments_come_as_far_as_the_device():
    for call in (norm, pack, matmul, scan):
        assert call() == R.EDEVICE, (call, R.last_error())
    assert norm(group=128) == R.EDEVICE and norm(group=0, weight=None) == R.EDEVICE
    assert norm(cols=20, group=20) == R.EDEVICE                        # a row of any multiple of 4
    assert norm(y=mem(1)) == R.EDEVICE                                 # in place
    assert norm(y=None) == R.EDEVICE and norm(q=None, q_scale=None) == R.EDEVICE and norm(res=None, gate=None, res_row=1) == R.EDEVICE
    assert norm(x_row=0) == R.EDEVICE                                  # one row for all
    assert norm(group=0, weight=mem(5)) == R.EDEVICE                   # no weight is read
    for kind in (R.I8_FROM_Q4K, R.I8_FROM_Q6K, R.I8_FROM_I8):
        assert pack(kind=kind) == R.EDEVICE
    assert pack(cols=528) == R.EDEVICE
    assert matmul(x_row=0) == R.EDEVICE and matmul(y_row=101) == R.EDEVICE
    assert scan(mode=R.SCAN_STATE, b=None, b_row=1 << 40) == R.EDEVICE
    assert scan(conv_b=None, dt_bias=None, skip=None) == R.EDEVICE and scan(most=1) == R.EDEVICE and scan(most=64) == R.EDEVICE
    assert scan(a_row=0) == R.EDEVICE and scan(x_row=8196) == R.EDEVICE


def test_no_rows_do_nothing():
    assert norm(rows=0) == R.OK and matmul(rows=0) == R.OK and scan(rows=0) == R.OK


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=(1 << 20) + 1), dict(cols=0), dict(cols=2046), dict(cols=16388), dict(group=8), dict(group=512),
    dict(group=96), dict(group=-1), dict(group=1024), dict(cols=2052, group=64, x_row=2052, res_row=2052, y_row=2052, q_row=2052),
    dict(x=None), dict(y=None, q=None), dict(q_scale=None), dict(x=mem(1) + 4), dict(res=mem(2) + 8), dict(weight=mem(3) + 4),
    dict(gate=mem(4) + 4), dict(y=mem(5) + 8), dict(q=mem(6) + 2), dict(q_scale=mem(7) + 1), dict(x_row=2050), dict(gate_row=2049),
    dict(res_row=2044), dict(y_row=1024), dict(q_row=2047), dict(q_row=2044), dict(x_row=1 << 33), dict(res=mem(1)), dict(y=mem(1), y_row=2052),
    dict(y=mem(1) + 16), dict(y=mem(2)), dict(y=mem(4) + 4096), dict(q=mem(5)), dict(q_scale=mem(6) + 64), dict(q=mem(3)),
    dict(res=mem(4)), dict(q_scale=mem(2) + 8192)])
def test_norm_refuses(kw):
    assert norm(**kw) == R.EINVAL, kw


@pytest.mark.parametrize("kw", [
    dict(rows=0), dict(rows=(1 << 20) + 1), dict(cols=0), dict(cols=24), dict(cols=65552), dict(data=None), dict(scale=None),
    dict(data=mem(1) + 8), dict(scale=mem(2) + 2)])
def test_weights_refused(kw):
    assert pack(**kw) == R.EINVAL and matmul(i8(**kw)) == R.EINVAL
    if "rows" in kw or "cols" in kw:
        assert R.lib().roaster_i8_bytes(kw.get("rows", 100), kw.get("cols", 512)) == 0


@pytest.mark.parametrize("kw", [
    dict(W=None), dict(kind=-1), dict(kind=4), dict(kind=R.I8_FROM_Q4K, cols=528), dict(kind=R.I8_FROM_Q6K, cols=128), dict(W=mem(3) + 4),
    dict(kind=R.I8_FROM_I8, W=mem(3) + 8), dict(W=mem(1)), dict(W=mem(1) - 16), dict(W=mem(2)), dict(scale=mem(1) + 4096)])
def test_pack_refuses(kw):
    assert pack(**kw) == R.EINVAL, kw


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=(1 << 20) + 1), dict(x=None), dict(x_scale=None), dict(y=None), dict(x=mem(3) + 8), dict(x_scale=mem(4) + 2),
    dict(y=mem(5) + 1), dict(x_row=520), dict(x_row=1 << 33), dict(y_row=99), dict(y_row=1 << 33), dict(y=mem(3)), dict(y=mem(4)),
    dict(y=mem(1) + 64), dict(y=mem(2) + 396)])
def test_matmul_refuses(kw):
    assert matmul(**kw) == R.EINVAL, kw


BAD_STATE = [dict(n_req=0), dict(n_req=2049), dict(k_heads=0), dict(k_heads=-1), dict(v_heads=0), dict(v_heads=24), dict(v_heads=272),
             dict(k_dim=96), dict(k_dim=256), dict(v_dim=32), dict(taps=1), dict(taps=5)]


@pytest.mark.parametrize("kw", BAD_STATE)
def test_state_refused(kw):
    s = state(**kw)
    assert scan(s) == R.EINVAL and R.lib().roaster_ssm_ws_bytes(64, 20, C.byref(s)) == 0


@pytest.mark.parametrize("kw", [dict(conv=None), dict(state=None), dict(conv=mem(1) + 8), dict(state=mem(2) + 4), dict(state=mem(1))])
def test_state_memory_refused(kw):
    assert scan(state(**kw)) == R.EINVAL


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=(1 << 18) + 1), dict(most=0), dict(most=65), dict(mode=2), dict(mode=-1), dict(x=None), dict(a=None), dict(b=None),
    dict(conv_w=None), dict(a_coef=None), dict(first=None), dict(row_pos=None), dict(out=None), dict(ws=None), dict(x=mem(3) + 8),
    dict(a=mem(4) + 2), dict(b=mem(5) + 1), dict(conv_w=mem(6) + 4), dict(conv_b=mem(7) + 2), dict(a_coef=mem(8) + 3), dict(dt_bias=mem(9) + 1),
    dict(skip=mem(10) + 2), dict(first=mem(11) + 2), dict(row_pos=mem(12) + 1), dict(out=mem(13) + 8), dict(ws=mem(14) + 8), dict(x_row=8190),
    dict(x_row=1 << 33), dict(a_row=1 << 33), dict(b_row=1 << 33), dict(out_row=4092), dict(out_row=4098), dict(ws_bytes=0), dict(out=mem(3)),
    dict(out=mem(1)), dict(out=mem(2) + 64), dict(out=mem(12)), dict(ws=mem(13)), dict(ws=mem(1) + 64), dict(out=mem(5)), dict(out=mem(8))])
def test_scan_refuses(kw):
    assert scan(**kw) == R.EINVAL, kw


def test_workspace_is_checked_and_grows():
    s = state()
    ws = lambda rows, most: R.lib().roaster_ssm_ws_bytes(rows, most, C.byref(s))  # noqa: E731
    sizes = [(0, 1), (1, 1), (64, 1), (64, 8), (64, 64), (2048, 64), (2048, 2048), (1 << 18, 1 << 18)]
    got = [ws(*z) for z in sizes]
    assert all(got) and got == sorted(got)
    assert ws(-1, 1) == 0 and ws(8, 9) == 0 and ws(8, 0) == 0 and ws((1 << 18) + 1, 1) == 0
    for rows, most in sizes[1:]:
        assert scan(rows=rows, most=most, ws_bytes=ws(rows, most) - 1) == R.EINVAL


def test_bytes_of_weights():
    assert R.lib().roaster_i8_bytes(1, 16) == 32 * 128 and R.lib().roaster_i8_bytes(33, 144) == 64 * 256
    assert R.lib().roaster_i8_bytes(1 << 20, 65536) == 1 << 36


@pytest.mark.parametrize("most", [1, 16, 64, 4096])
@pytest.mark.parametrize("n_req", [1, 8, 2048])
def test_a_workspace_for_no_rows(n_req, most):
    """A step without rows is a good one, whatever `most`: 0 bytes would say that its arguments are bad."""
    assert R.lib().roaster_ssm_ws_bytes(0, most, C.byref(state(n_req=n_req))) > 0
