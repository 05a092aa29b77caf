"""Gated recurrence and its backward pass against the formula token by token in
64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from hephaestus_amd import Layout, StridedView
from layer_reference import EPS32, as_float64, padded, rounded, vector
from training_reference import TYPES, gated_recurrence, gated_recurrence_backward, near

pytestmark = pytest.mark.gpu

# Tiles of 128 and 64 tokens, 64 and 128 channels; parts where channels are few.
SIZES = [(1, 1, 1), (2, 1, 7), (3, 2, 64), (1, 7, 130), (2, 8, 65), (1, 32, 128), (2, 33, 3), (1, 64, 200), (2, 65, 96),
         (1, 127, 66), (3, 128, 64), (1, 129, 129), (2, 300, 5), (1, 1000, 40), (1, 4097, 6), (70, 40, 260),
         (200, 130, 64)]


def operands(t, batch, tokens, channels, seed=0):
    rng = np.random.default_rng(seed)
    gate = rounded(rng.normal(size=(batch, tokens, channels)) + rng.uniform(-2, 7, channels), t)
    x, dy = rounded(rng.normal(size=(batch, tokens, channels)), t), rounded(rng.normal(size=(batch, tokens, channels)) * 0.01, t)
    first, dlast = rng.normal(size=(2, batch, channels)).astype(np.float32)
    return gate, x, dy, first, dlast * np.float32(0.01)


def forward(device, gate, x, first, lengths=None, **place):
    vz, vx = padded(device, gate, **place)[0], padded(device, x, **place)[0]
    vh, read_h = padded(device, rounded(np.full(x.shape, 9.0), x.dtype), **place)
    vs, read_s = padded(device, np.full((x.shape[0], x.shape[2]), 9, np.float32))
    hx.RocmRecurrenceOps().gated_recurrence_into(
        device, vz, vx, vh, state_in=None if first is None else padded(device, first, 3)[0], state_out=vs,
        lengths=None if lengths is None else vector(device, np.asarray(lengths, np.uint32)))
    device.synchronize()
    return {"h": read_h(), "last": read_s()}


def backward(device, gate, x, h, dy, first, dlast, lengths=None, **place):
    views = [padded(device, v, **place)[0] for v in (gate, x, h, dy)]
    vz, read_z = padded(device, rounded(np.full(x.shape, 9.0), x.dtype), **place)
    vx, read_x = padded(device, rounded(np.full(x.shape, 9.0), x.dtype), **place)
    vs, read_s = padded(device, np.full((x.shape[0], x.shape[2]), 9, np.float32), 1)
    hx.RocmRecurrenceOps().gated_recurrence_backward_into(
        device, *views, vz, vx, state_in=None if first is None else padded(device, first)[0],
        grad_state_out=None if dlast is None else padded(device, dlast, 2)[0], grad_state_in=vs,
        lengths=None if lengths is None else vector(device, np.asarray(lengths, np.uint32)))
    device.synchronize()
    return {"dgate": read_z(), "dx": read_x(), "dfirst": read_s()}


def check(got, expected):
    value, bound = expected
    for name in got:
        near(got[name], value[name], bound[name], name)


def check_both(device, gate, x, dy, first, dlast, lengths=None, **place):
    got = forward(device, gate, x, first, lengths, **place)
    check(got, gated_recurrence(gate, x, first, lengths))
    check(backward(device, gate, x, got["h"], dy, first, dlast, lengths, **place),
          gated_recurrence_backward(gate, x, got["h"], dy, first, dlast, lengths))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,tokens,channels", SIZES)
def test_sizes(device, dtype, batch, tokens, channels):
    check_both(device, *operands(TYPES[dtype], batch, tokens, channels, tokens + channels))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 20, 700])
def test_without_states(device, dtype, tokens):
    gate, x, dy, _, _ = operands(TYPES[dtype], 2, tokens, 70, tokens)
    check_both(device, gate, x, dy, None, None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,channels", [(5, 64), (200, 33), (900, 20), (130, 5000)])
def test_lengths(device, dtype, tokens, channels):
    """None, one, some and all tokens; what lies past a sequence's end is not read
    into a result and gives zeros, and a length past the end is the end."""
    gate, x, dy, first, dlast = operands(TYPES[dtype], 6, tokens, channels, tokens)
    lengths = [0, 1, tokens // 2, tokens - 1, tokens, tokens + 5]
    nan = rounded(np.array([np.nan]), x.dtype)[0]
    for b, n in enumerate(lengths):
        for v in (gate, x, dy):
            v[b, n:] = nan
    got = forward(device, gate, x, first, lengths)
    check(got, gated_recurrence(gate, x, first, lengths))
    assert np.array_equal(got["last"][0], first[0])
    h = got["h"].copy()
    for b, n in enumerate(lengths):
        assert not as_float64(h[b, n:]).any()
        h[b, n:] = nan
    back = backward(device, gate, x, h, dy, first, dlast, lengths)
    check(back, gated_recurrence_backward(gate, x, h, dy, first, dlast, lengths))
    assert np.array_equal(back["dfirst"][0], dlast[0])
    for b, n in enumerate(lengths):
        assert not as_float64(back["dx"][b, n:]).any() and not as_float64(back["dgate"][b, n:]).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("place", [{"strides_pad": 1}, {"strides_pad": 2, "offset": 1}, {"offset": 2},
                                   {"order": (1, 0, 2)}, {"order": (1, 0, 2), "strides_pad": 6}])
@pytest.mark.parametrize("tokens,channels", [(1, 130), (40, 66), (260, 64)])
def test_strides(device, dtype, place, tokens, channels):
    check_both(device, *operands(TYPES[dtype], 3, tokens, channels, 5), **place)


@pytest.mark.parametrize("dtype", TYPES)
def test_gate_and_input_in_one_row(device, dtype):
    """Both halves of a projection's rows, and their gradients beside each other."""
    t, (b, n, c) = TYPES[dtype], (2, 150, 64)
    gate, x, dy, first, dlast = operands(t, b, n, c, 8)
    both = device.upload(np.concatenate([gate, x], axis=2))
    out = device.upload(rounded(np.zeros((b, n, 2 * c)), t))
    halves = [[StridedView(buf, Layout.try_new([b, n, c], [n * 2 * c, 2 * c, 1], part * c)) for part in range(2)]
              for buf in (both, out)]
    vh, read_h = padded(device, rounded(np.zeros((b, n, c)), t))
    ops = hx.RocmRecurrenceOps()
    ops.gated_recurrence_into(device, *halves[0], vh)
    ops.gated_recurrence_backward_into(device, *halves[0], vh, padded(device, dy)[0], *halves[1])
    device.synchronize()
    check({"h": read_h()}, gated_recurrence(gate, x))
    value, bound = gated_recurrence_backward(gate, x, read_h(), dy)
    got = device.download_owned(out).reshape(b, n, 2 * c)
    near(got[:, :, :c], value["dgate"], bound["dgate"], "dgate")
    near(got[:, :, c:], value["dx"], bound["dx"], "dx")


@pytest.mark.parametrize("dtype", TYPES)
def test_state_in_place_token_by_token(device, dtype):
    """A prompt and then single tokens, the state where it was: as all at once."""
    t, steps = TYPES[dtype], 4
    gate, x, _, first, _ = operands(t, 3, 300 + steps, 70, 2)
    state, read = padded(device, first, 5)
    ops, parts = hx.RocmRecurrenceOps(), []
    for lo, hi in [(0, 300)] + [(300 + i, 301 + i) for i in range(steps)]:
        vh, read_h = padded(device, rounded(np.zeros((3, hi - lo, 70)), t))
        ops.gated_recurrence_into(device, padded(device, gate[:, lo:hi])[0], padded(device, x[:, lo:hi])[0], vh,
                                  state_in=state, state_out=state)
        device.synchronize()
        parts.append(read_h())
    check({"h": np.concatenate(parts, 1), "last": read()}, gated_recurrence(gate, x, first))


@pytest.mark.parametrize("tokens", [1, 20, 500])
def test_gates_that_are_shut_or_open(device, tokens):
    """f is 0 or 1 to the bit where the gate is infinite: a reset forgets whatever
    finite state there was, an open gate keeps it."""
    gate, x, dy, first, dlast = operands(np.float32, 1, tokens, 8, 1)
    first[:] = 1e30
    gate[:, 0] = -np.inf
    check_both(device, gate, x, dy, first, dlast)
    gate[:] = np.inf
    got = forward(device, gate, x, first)
    assert np.array_equal(got["last"], first) and np.array_equal(got["h"], np.broadcast_to(first[:, None], x.shape))
    back = backward(device, gate, x, got["h"], dy, first, dlast)
    assert not back["dx"].any() and not back["dgate"].any()


@pytest.mark.parametrize("tokens", [20, 600])
def test_values_that_are_no_numbers_stay_in_their_channels(device, tokens):
    gate, x, dy, first, dlast = operands(np.float32, 2, tokens, 9, 1)
    x[0, 7, 3], gate[1, 4, 5] = np.nan, np.nan
    got = forward(device, gate, x, first)
    bad = np.zeros(x.shape, bool)
    bad[0, 7:, 3] = bad[1, 4:, 5] = True
    assert np.isnan(got["h"][bad]).all()
    clean_gate, clean_x = np.where(np.isnan(gate), 0, gate), np.where(np.isnan(x), 0, x)
    value, bound = gated_recurrence(clean_gate, clean_x, first)
    near(got["h"][~bad], value["h"][~bad], bound["h"][~bad], "h")


def test_long_memory_in_f32(device):
    """A state that all of 20000 tokens matter to, f within 2^-15 of 1: what a factor's
    own rounding would leave, 2^-25 a token, does not add up."""
    rng = np.random.default_rng(3)
    gate = np.full((1, 20000, 16), 10.4, np.float32)
    x = rng.normal(size=gate.shape).astype(np.float32) + 1
    dy = rng.normal(size=gate.shape).astype(np.float32) + 1
    got = forward(device, gate, x, None)
    f, rest = 1 / (1 + np.exp(-gate[0, 0].astype(np.float64))), 1 / (1 + np.exp(gate[0, 0].astype(np.float64)))
    left = f[None] ** np.arange(19999, -1, -1)[:, None]
    want = (left * rest * x[0].astype(np.float64)).sum(0)
    # Each token's sum is rounded once, 2^-25 of the state at random, over 20000 tokens.
    assert np.abs(got["last"][0] - want).max() <= 6 * 2.0**-25 * np.sqrt(20000) * np.abs(want).max()
    back = backward(device, gate, x, got["h"], dy, None, None)
    want = (f[None] ** np.arange(1, 20001)[:, None] * dy[0].astype(np.float64)).sum(0)
    assert np.abs(back["dfirst"][0] - want).max() <= 6 * 2.0**-25 * np.sqrt(20000) * np.abs(want).max()


def test_empty(device):
    f = np.float32
    none = device.alloc_zeroed(f, 0)
    for shape in ([0, 4, 5], [2, 4, 0]):
        v = StridedView(none, Layout.c_contiguous(shape))
        hx.RocmRecurrenceOps().gated_recurrence_into(device, v, v, v)
    # No tokens: the state passes through.
    v = StridedView(none, Layout.c_contiguous([2, 0, 5]))
    first = np.arange(10, dtype=f).reshape(2, 5)
    vs, read = padded(device, np.zeros((2, 5), f))
    hx.RocmRecurrenceOps().gated_recurrence_into(device, v, v, v, state_in=padded(device, first)[0], state_out=vs)
    device.synchronize()
    assert np.array_equal(read(), first)


@pytest.mark.parametrize("tokens", [3, 150])
def test_gradient_against_differences(device, tokens):
    """Of L = Σ dy·h + Σ dlast·last, by two evaluations in 64 bits."""
    gate, x, dy, first, dlast = operands(np.float32, 2, tokens, 6, 4)
    got = forward(device, gate, x, first)
    back = backward(device, gate, x, got["h"], dy, first, dlast)
    rng = np.random.default_rng(1)

    def loss(z, u, s):
        f = 1 / (1 + np.exp(-z))
        total, state = 0.0, s
        for t in range(tokens):
            state = f[:, t] * state + (1 - f[:, t]) * u[:, t]
            total += (dy[:, t].astype(np.float64) * state).sum()
        return total + (dlast.astype(np.float64) * state).sum()

    base = [v.astype(np.float64) for v in (gate, x, first)]
    for i, name in enumerate(("dgate", "dx", "dfirst")):
        way, h = rng.normal(size=base[i].shape), 1e-4
        up, down = [list(base), list(base)]
        up[i], down[i] = base[i] + h * way, base[i] - h * way
        slope = (loss(*up) - loss(*down)) / (2 * h)
        size = np.abs(back[name].astype(np.float64) * way).sum()
        assert abs((back[name].astype(np.float64) * way).sum() - slope) <= 1e-5 * size + 1e-7


def test_runs_repeat_to_the_bit(device):
    gate, x, dy, first, dlast = operands(np.float32, 1, 3000, 100, 4)
    h = forward(device, gate, x, first)
    back = backward(device, gate, x, h["h"], dy, first, dlast)
    for _ in range(2):
        again = forward(device, gate, x, first)
        assert all(np.array_equal(h[k], again[k]) for k in h)
        again = backward(device, gate, x, h["h"], dy, first, dlast)
        assert all(np.array_equal(back[k], again[k]) for k in back)


def test_offsets_past_32_bits(device):
    """Tokens 2^32 bytes and more into a view: single tokens far apart, read by two
    sequences of one pool."""
    t, far = hx.bfloat16, (1 << 31) + 64  # elements between the two tokens
    pool = device.alloc_uninitialized(t, far + 64)
    view = StridedView(pool, Layout.try_new([1, 2, 64], [0, far, 1]))
    gate, x, _, first, _ = operands(t, 1, 2, 64, 3)
    one = np.empty((2, 64), t)
    for i in range(2):
        one[i] = x[0, i]
        hx.RocmDevice.write_sub_buffer(device, pool, i * far, x[0, i])
    vh, read = padded(device, rounded(np.zeros((1, 2, 64)), t))
    hx.RocmRecurrenceOps().gated_recurrence_into(device, padded(device, gate)[0], view, vh,
                                                 state_in=padded(device, first)[0])
    device.synchronize()
    check({"h": read()}, gated_recurrence(gate, x, first))
