"""Linear attention against its recurrence in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from layer_reference import EPS16, EPS32, as_float64, linear_attention, padded, rounded, vector

pytestmark = pytest.mark.gpu

TYPES = {"f32": np.float32, "bf16": hx.bfloat16}
ORDERS = {"tokens": None, "heads": (0, 2, 1, 3), "tokens first": (1, 0, 2, 3)}


def operands(dtype, batch, tokens, heads, kv_heads, dk, dv, seed=0):
    rng = np.random.default_rng([seed, batch, tokens, heads, kv_heads, dk, dv])
    q = rounded(rng.normal(size=(batch, tokens, heads, dk)), dtype)
    k = rounded(rng.normal(size=(batch, tokens, kv_heads, dk)), dtype)
    v = rounded(rng.normal(size=(batch, tokens, kv_heads, dv)), dtype)
    decay = np.log1p(-(2.0 ** -rng.uniform(1, 10, heads))).astype(np.float32)
    return q, k, v, decay, rng.normal(size=(batch, heads, dk, dv)).astype(np.float32) * 2


def run(device, q, k, v, decay, state=None, lengths=None, *, scale=None, order=None, pad=0, offset=0, prepared=False,
        keep_state=True):
    views = [padded(device, x, pad, offset, order)[0] for x in (q, k, v)]
    shape = (*q.shape[:3], v.shape[3])
    vo, read_o = padded(device, rounded(np.full(shape, 5.0), q.dtype), pad, offset, order)
    states = (q.shape[0], q.shape[2], q.shape[3], v.shape[3])
    vs, read_s = padded(device, np.full(states, 5.0, np.float32), pad, offset)
    args = (device, *views, vector(device, decay), vo)
    more = {"scale": scale, "state_in": None if state is None else padded(device, state, pad and 4, offset)[0],
            "state_out": vs if keep_state else None,
            "lengths": None if lengths is None else vector(device, np.asarray(lengths, np.uint32))}
    if prepared:
        plan = hx.RocmLinearAttentionOps().prepare_linear_attention(*args, **more)
        plan.dispatch()
        plan.dispatch()
    else:
        hx.RocmLinearAttentionOps().linear_attention_into(*args, **more)
    device.synchronize()
    return read_o(), read_s() if keep_state else None


def check(q, k, v, decay, state, lengths, got, scale=None):
    scale = np.float32(q.shape[3] ** -0.5 if scale is None else scale)
    want, last, size, last_size = linear_attention(q, k, v, decay, float(scale), state, lengths)
    # In f32: the decay's rounding at each token, the sum over dk, a few more.
    # In bf16 every score and every element of a state that a query meets is
    # rounded once, and the output once.
    steps = (3 * q.shape[1] + q.shape[3] + 16) * EPS32
    bound = steps * size
    if q.dtype == hx.bfloat16:
        bound = bound + EPS16 * (size + np.abs(want)) * (1 + 2.0**-8)
    off = np.abs(as_float64(got[0]) - want)
    assert np.all(off <= bound), (np.max(off - bound), np.unravel_index(np.argmax(off - bound), off.shape))
    if got[1] is not None:
        off = np.abs(got[1] - last)
        assert np.all(off <= steps * last_size), np.unravel_index(np.argmax(off - steps * last_size), off.shape)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 2, 3, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 200])
def test_lengths_of_a_prompt(device, dtype, tokens):
    ops = operands(TYPES[dtype], 2, tokens, 3, 3, 32, 48)
    check(*ops, None, run(device, *ops))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 70])
@pytest.mark.parametrize("dk,dv", [
    (1, 1), (3, 5), (8, 8), (16, 16), (17, 31), (32, 32), (37, 53), (64, 64), (80, 96), (96, 80), (100, 128),
    (128, 128), (128, 130), (129, 64), (160, 33), (200, 100), (256, 128), (256, 256), (64, 300)])
def test_widths_of_heads(device, dtype, tokens, dk, dv):
    ops = operands(TYPES[dtype], 1, tokens, 2, 1, dk, dv)
    check(*ops, None, run(device, *ops))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 5, 150])
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 16), (1, 3)])
def test_orders_strides_and_offsets(device, dtype, tokens, order, pad, offset):
    ops = operands(TYPES[dtype], 3, tokens, 4, 2, 40, 64)
    check(*ops, None, run(device, *ops, order=ORDERS[order], pad=pad, offset=offset, prepared=True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (6, 3), (8, 1), (5, 5), (12, 4)])
def test_shared_heads(device, dtype, heads, kv_heads):
    for tokens in (1, 90):
        ops = operands(TYPES[dtype], 2, tokens, heads, kv_heads, 64, 64)
        check(*ops, None, run(device, *ops))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_state", [False, True])
@pytest.mark.parametrize("tokens,lengths", [(200, [200, 0, 1, 64, 63, 65, 199, 128]), (1, [1, 0]), (7, [3, 0, 7, 900]),
                                            (70, [0, 0, 0])])
def test_lengths_of_sequences(device, dtype, with_state, tokens, lengths):
    """Sequences of no tokens and one, and counts past the end; the rows past
    a length hold NaN, which must not be read."""
    q, k, v, decay, state = operands(TYPES[dtype], len(lengths), tokens, 2, 1, 64, 48, 3)
    nan = rounded(np.full(1, np.nan), TYPES[dtype])[0]
    for b, count in enumerate(lengths):
        for x in (q, k, v):
            x[b, count:] = nan
    state = state if with_state else None
    got = run(device, q, k, v, decay, state, lengths)
    for b, count in enumerate(lengths):
        assert not as_float64(got[0])[b, count:].any()
    clean = [x.copy() for x in (q, k, v)]
    for b, count in enumerate(lengths):
        for x in clean:
            x[b, count:] = rounded(np.zeros(1), TYPES[dtype])[0]
    check(*clean, decay, state, lengths, got)
    for b, count in enumerate(lengths):
        if count == 0:
            assert np.array_equal(got[1][b], np.zeros_like(got[1][b]) if state is None else state[b])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 150])
def test_decays_at_their_ends(device, dtype, tokens):
    """No decay, none kept, and heads that forget within a token."""
    q, k, v, _, state = operands(TYPES[dtype], 1, tokens, 6, 6, 32, 32)
    decay = np.array([0.0, -np.inf, -1e-7, -5.0, -80.0, -1e30], np.float32)
    got = run(device, q, k, v, decay, state)
    check(q, k, v, decay, state, None, got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 130])
def test_no_state_in_or_out_and_a_scale(device, dtype, tokens):
    q, k, v, decay, _ = operands(TYPES[dtype], 2, tokens, 2, 2, 48, 48)
    got = run(device, q, k, v, decay, keep_state=False, scale=-2.5)
    check(q, k, v, decay, None, None, got, scale=-2.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,tokens,heads", [(1, 1500, 1), (2, 700, 2), (1, 4100, 2)])
def test_long_prompts(device, dtype, batch, tokens, heads):
    """Few heads and many tokens: the prompt is split and joined."""
    ops = operands(TYPES[dtype], batch, tokens, heads, 1, 16, 16)
    check(*ops, None, run(device, *ops, prepared=True))
    lengths = [tokens // 3, tokens][:batch]
    q, k, v, decay, state = ops
    check(q, k, v, decay, state, lengths, run(device, *ops, lengths))


@pytest.mark.parametrize("dtype", TYPES)
def test_state_carries_a_prompt_over(device, dtype):
    """A prompt, then single tokens with the state updated in place, equals the
    whole at once."""
    q, k, v, decay, state = operands(TYPES[dtype], 2, 80, 3, 3, 64, 64, 9)
    vs, read = padded(device, state)
    ops, outs = hx.RocmLinearAttentionOps(), []
    cuts = [0, 70, *range(71, 81)]
    for lo, hi in zip(cuts, cuts[1:]):
        views = [padded(device, np.ascontiguousarray(x[:, lo:hi]))[0] for x in (q, k, v)]
        vo, read_o = padded(device, rounded(np.zeros((2, hi - lo, 3, 64)), q.dtype))
        ops.linear_attention_into(device, *views, vector(device, decay), vo, state_in=vs, state_out=vs)
        device.synchronize()
        outs.append(as_float64(read_o()))
    got = np.concatenate(outs, 1)
    check(q, k, v, decay, state, None, (got if q.dtype == np.float32 else rounded(got, q.dtype), read()))


def test_no_tokens_and_no_heads(device):
    q, k, v, decay, state = operands(np.float32, 2, 0, 3, 3, 16, 16)
    _, last = run(device, q, k, v, decay, state)
    assert np.array_equal(last, state)
    got, _ = run(device, *operands(np.float32, 2, 4, 0, 0, 16, 16)[:4], keep_state=False)
    assert got.shape == (2, 4, 0, 16)
    got, _ = run(device, *operands(np.float32, 2, 4, 2, 2, 0, 16)[:4], keep_state=False, scale=1.0)
    assert not got.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_stay_with_their_head_and_time(device, dtype):
    q, k, v, decay, state = operands(TYPES[dtype], 1, 100, 2, 2, 32, 32)
    bad = rounded(np.array([np.inf]), TYPES[dtype])[0]
    v[0, 60, 1, 3] = bad
    got, last = run(device, q, k, v, decay, state)
    got = as_float64(got)
    assert np.isfinite(got[:, :, 0]).all() and np.isfinite(np.delete(got[:, :, 1], 3, -1)).all()
    assert np.isfinite(got[:, :60, 1]).all()
    assert not np.isfinite(got[:, 60:, 1, 3]).any()
    assert np.isfinite(last[:, 0]).all() and not np.isfinite(last[:, 1, :, 3]).any()
