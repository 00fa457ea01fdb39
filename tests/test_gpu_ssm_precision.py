"""How near roaster_ssm_scan's prompts, taken 64 tokens at a time, come to the recurrence in 64 bits
where a bound of the state could leave the state behind: long prompts without decay, values far above
the ones that follow, steps and values that peak at different tokens, decays that wipe a state out.

Each is held to the plain recurrence in f32 on the same inputs: the error over a span of tokens is at most
eight of its errors (operands of 22 bits to f32's 24, whose products leave out up to another 2^-22) and
FINE times the largest |v| and row of the state in the span.  FINE: an operand's lowest bit is 2^-30 of those,
and a row's error sums up to 128 elements' or 64 tokens', which do not all point one way: 16 of them."""
import numpy as np
import pytest

import roaster_amd as R
from attn_util import sync
from gpu_util import log
from mixer_util import Scan, ScanCall, check_scan, scan_oracle, sigmoid

pytestmark = pytest.mark.gpu
DELTA, STATE = R.SCAN_DELTA, R.SCAN_STATE
FINE = 16 * 2.0 ** -30


def recurrence(s, t):
    """Request 0's outputs [rows][v_heads][v_dim], states of each 64th token and, by value head, the largest
    |v| (STATE: |dt v| |k|) and row of the state of each 64 tokens, every step in type t."""
    n, rep, nk = s.new[0], s.vh // s.kh, s.kh * s.kd
    f = lambda v: v.astype(t)  # noqa: E731
    x, w = f(s.x[:n, :s.C]), f(s.conv_w)
    c = np.zeros_like(x) if s.conv_b is None else np.broadcast_to(f(s.conv_b), x.shape).copy()
    for j in range(s.taps):
        back = s.taps - 1 - j
        c[back:] += x[:n - back] * w[:, j]
    c = (c * sigmoid(c)).astype(t)
    q, k, v = c[:, :nk].reshape(n, s.kh, s.kd), c[:, nk:2 * nk].reshape(n, s.kh, s.kd), c[:, 2 * nk:].reshape(n, s.vh, s.vd)
    a = f(s.a[:n, :s.vh]) + (t(0) if s.dt_bias is None else f(s.dt_bias))
    dt = np.maximum(a, t(0)) + np.log1p(np.exp(-np.abs(a)))
    decay = np.exp(f(s.a_coef) * dt)
    if s.mode == DELTA:
        q, k = (z / np.sqrt((z * z).sum(axis=2, keepdims=True) + t(s.eps)) for z in (q, k))
        gain = sigmoid(f(s.b[:n, :s.vh])).astype(t)
    else:
        gain = dt
    q, k = np.repeat(q * t(s.scale), rep, axis=1), np.repeat(k, rep, axis=1)
    out, S = np.empty((n, s.vh, s.vd), t), np.zeros((s.vh, s.vd, s.kd), t)
    size = []
    for i in range(n):
        S *= decay[i][:, None, None]
        u = v[i]
        if s.mode == DELTA:
            u = u - np.matmul(S, k[i][..., None])[..., 0]
        u = gain[i][:, None] * u
        S += u[..., None] * k[i][:, None]
        out[i] = np.matmul(S, q[i][..., None])[..., 0]
        if i % 64 == 63 or i == n - 1:
            at = slice(i // 64 * 64, i + 1)
            b = np.abs(v[at]) if s.mode == DELTA else np.abs(gain[at][..., None] * v[at]) * np.linalg.norm(k[at], axis=2)[..., None]
            size.append(np.maximum(b.max(axis=0), np.linalg.norm(S, axis=2)))
    return out if s.skip is None else out + f(s.skip)[:, None] * v, S, np.array(size)


def compare(s, spans):
    """The prompt of s, which begins at position 0, over spans of tokens: errors of its outputs, and of its states at the end."""
    call = ScanCall(s)
    R.check(call.call(), "scan")
    sync()
    out, _, state = call.got()
    o, S, size = recurrence(s, np.float64)
    o32, S32, _ = recurrence(s, np.float32)
    worst = []
    for lo, hi in spans:
        at = slice(lo, hi)
        top = size[max(0, lo // 64 - 1):-(-hi // 64)].max(axis=0) * abs(s.scale) * (1 if s.mode == DELTA else 16)
        err, plain = np.abs(out[at] - o[at]).max(axis=0), np.abs(o32[at] - o[at]).max()
        lim = 8 * plain + FINE * top
        log(f"tokens {lo} .. {hi}: error {err.max():.2e}, in f32 {plain:.2e}, outputs up to {np.abs(o[at]).max():.2e}, share of the limit "
            f"{(err / lim).max():.2g}")
        worst.append((err / lim).max())
    err, plain = np.linalg.norm(state[0] - S, axis=2), np.linalg.norm(S32 - S, axis=2).max()
    lim = 8 * plain + FINE * size[-2:].max(axis=0)
    log(f"state: error {err.max():.2e}, in f32 {plain:.2e}, share {(err / lim).max():.2g}")
    assert max(worst) <= 1 and np.all(err <= lim)


def slow(rng, n, mode, coef=-2e-4, **kw):
    """A prompt whose heads hardly decay: log decays of about 0.05 * coef a token."""
    s = Scan(rng, [n], [0], mode, 1, 2, 128, 64, dt_bias=False, skip=False, **kw)
    s.a[:], s.a_coef[:] = -3 + 0.1 * s.a, coef
    return s


@pytest.mark.parametrize("coef", [-2e-4, 0.0])
@pytest.mark.parametrize("early,by", [(1, 1e6), (64, 1e5)])
def test_large_values_at_the_beginning(early, by, coef):
    """Keys of one direction after the other, so that the correction takes the large values out of the state within a thousand
    tokens; those behind have the precision of their own values."""
    s = slow(np.random.default_rng(31), 4096, DELTA, coef, taps=2, bias=False)
    s.x[:early, 256:] *= np.float32(by)
    s.conv_w[:, 0], s.conv_w[:, 1] = 0, 1
    s.x[:, 128:256] = 0.1 * s.x[:, 128:256] - 8
    s.x[np.arange(4096), 128 + np.arange(4096) % 128] += 16
    s.b[:] = 2 + 0.1 * s.b
    compare(s, [(0, 256), (3200, 4096)])


@pytest.mark.parametrize("early,by", [(1, 1e6), (64, 1e5)])
def test_large_values_that_decay(early, by):
    """Without the correction: e^-0.01 a token."""
    s = slow(np.random.default_rng(32), 4096, STATE, -0.2)
    s.x[:early, 256:] *= np.float32(by)
    compare(s, [(0, 256), (3200, 4096)])


@pytest.mark.parametrize("mode", [DELTA, STATE])
@pytest.mark.parametrize("at", [64, 100, 127])
def test_a_large_value_in_the_middle(mode, at):
    """It takes bits from the 64 tokens that it is taken with and from the next 64, from none before them."""
    s = slow(np.random.default_rng(38), 256, mode, -2e-4, taps=2, bias=False)
    s.conv_w[256:, 0], s.conv_w[256:, 1] = 0, 1
    s.x[at, 256:] *= np.float32(1e6)
    compare(s, [(0, 64), (64, at), (at, 128), (128, 192)] if at > 64 else [(0, 64), (64, 128), (128, 192)])


@pytest.mark.parametrize("mode", [DELTA, STATE])
def test_a_long_prompt_without_decay(mode):
    compare(slow(np.random.default_rng(33), 20000, mode, 0.0), [(0, 64), (19000, 20000)])


@pytest.mark.parametrize("coef", [-1e-7, -0.01])
def test_steps_and_values_that_peak_at_different_tokens(coef):
    """Every other token has a step of about 100 and a value of 0.01, those between a step of 1e-4 and values of up to 1e4."""
    s = slow(np.random.default_rng(34), 2048, STATE, coef, taps=2, bias=False)
    s.conv_w[256:, 0], s.conv_w[256:, 1] = 0, 1
    s.a[::2], s.a[1::2] = 100, np.float32(np.log(1e-4))
    s.x[::2, 256:] *= np.float32(0.01)
    s.x[1::2, 256:] *= np.float32(1e4)
    compare(s, [(0, 64), (1024, 2048)])


@pytest.mark.parametrize("mode", [DELTA, STATE])
@pytest.mark.parametrize("a", [300.0, 1e13, 1e17, 1e20, 1e36])
def test_a_token_that_wipes_the_state_out(mode, a):
    """A step of 1e13 and more leaves nothing of the state before it; the tokens behind it decay as ever.  STATE: without a
    value of its own, which such a step would put far above all others."""
    s = Scan(np.random.default_rng(35), [100, 40], [0, 4], mode, 2, 4, 64, 64, taps=2, bias=False, dt_bias=False)
    s.a[:], s.a_coef[:] = 0.1 * s.a - 2, -0.8                # e^-0.1 a token
    for at in (9, 10, 70, 108):
        s.a[at] = np.float32(a)
        if mode == STATE:
            s.x[at - 1:at + 1, 2 * 2 * 64:] = 0
    call = ScanCall(s)
    R.check(call.call(), "scan")
    sync()
    with np.errstate(over="ignore"):
        want = scan_oracle(s)
    log(check_scan(call.got(), want))


@pytest.mark.parametrize("mode", [DELTA, STATE])
def test_roundings_do_not_lean_to_one_side(mode):
    """What the products of operands in two parts leave out must not have the product's sign: the errors' mean along the outputs.
    The part of it that f32 itself has is that of constants (log2 e is off by 2^-26 of itself, in exponentials of about -2 .. 2)
    and of the reciprocal's last bit: below 2^-24 together; what is left of a million roundings that go either way is far
    below.  With high parts cut off a single product leans by (2^-11 * 0.7)^2, 2^-23, and outputs come through three in a row."""
    s = Scan(np.random.default_rng(36), [2048], [0], mode, 1, 4, 128, 128, skip=False)
    call = ScanCall(s)
    R.check(call.call(), "scan")
    sync()
    out = call.got()[0].astype(np.float64)
    o, _, _ = recurrence(s, np.float64)
    lean = ((out - o) * o).sum(axis=(0, 2)) / (o * o).sum(axis=(0, 2))
    log("errors along the outputs:", lean, "all of them:", np.linalg.norm(out - o) / np.linalg.norm(o))
    assert np.all(np.abs(lean) <= 2.0 ** -23)


@pytest.mark.parametrize("new", [[2, 1], [70, 33]])
def test_vectors_whose_squares_pass_the_range_are_zeros(new):
    """Key head 0's keys of one row and key head 1's queries of another are above 1e19: as if they were zeros, in both kernels."""
    s = Scan(np.random.default_rng(37), new, [0, 4], DELTA, 2, 4, 128, 128, taps=2, bias=False)
    s.conv_w[:512, 0], s.conv_w[:512, 1] = 0, 1
    rows = (new[0] - 1, new[0])
    parts = (slice(256, 384), slice(128, 256))
    for row, part in zip(rows, parts):
        s.x[row, part] = 0                                 # silu(0) = 0
    want = scan_oracle(s)
    for row, part in zip(rows, parts):
        s.x[row, part] = np.float32(3e19)
    call = ScanCall(s)
    R.check(call.call(), "scan")
    sync()
    out, conv, state = call.got()
    assert np.all(np.abs(out - want[0]) <= want[3] + 1e-30)
    assert np.all(np.linalg.norm(state - want[2], axis=3) <= want[4] + 1e-30)
