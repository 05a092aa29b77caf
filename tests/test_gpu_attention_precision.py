"""How many bits a prompt keeps: linear attention in chunks against closed forms in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from layer_reference import EPS16, EPS32, as_float64, linear_attention, padded
from test_gpu_layer_forms import by_pairs
from test_gpu_linear_attention import operands, run

pytestmark = pytest.mark.gpu


# Both sides of a chunk, of eight waves and four, and a prompt that is cut.
@pytest.mark.parametrize("tokens,heads,dk,dv", [
    (9, 2, 128, 128), (64, 3, 64, 64), (70, 3, 64, 64), (200, 2, 128, 128), (130, 2, 96, 80), (130, 2, 37, 53),
    (100, 2, 256, 64), (1300, 1, 64, 64), (1300, 1, 128, 128)])
def test_bf16_prompts_round_once(device, tokens, heads, dk, dv):
    """Outputs of bf16 prompts are f32 sums rounded once, as those of single
    tokens are."""
    q, k, v, decay, state = operands(hx.bfloat16, 2, tokens, heads, 1, dk, dv, 21)
    got = as_float64(run(device, q, k, v, decay, state)[0])
    want, _, size, _ = linear_attention(q, k, v, decay, float(np.float32(dk ** -0.5)), state)
    # Terms: two bf16 terms hold a score, and an element of a state, to 2^-15.
    # Sums: three roundings of the state for each chunk of 64 tokens, the sum
    # over dk, that over a chunk, and some for weights and scale.
    inner = 2 * 2.0**-15 + (3 * tokens / 64 + dk + 64 + 32) * EPS32
    assert np.all(np.abs(got - want) <= inner * size + EPS16 * (np.abs(want) + inner * size))
    # In the norm, an error apart from the last rounding adds its square to that
    # of the rounding: 2^-15 against 2^-10 or more.
    rounding = as_float64(hx.bfloat16_from_float32(want.astype(np.float32))) - want
    assert np.linalg.norm(got - want) <= 1.02 * np.linalg.norm(rounding)


def drifting_decays(rng, heads, chunk):
    """Log decays whose factor over a chunk, as a float, is too small by most of
    half a unit: 2^-25, relative."""
    found = []
    while len(found) < heads:
        g = rng.uniform(-0.1 / chunk, -0.02 / chunk, 4096).astype(np.float32)
        d = np.exp(g.astype(np.float64) * chunk)
        found.extend(g[(d - d.astype(np.float32)) / d >= 0.7 * 2.0**-25])
    return np.array(found[:heads], np.float32)


def bias(got, want):
    return float(np.vdot(got.astype(np.float64) - want, want) / np.vdot(want, want))


# Few tokens of 260 heads, so that a prompt is not cut and its chunks follow one
# another in a block.  Roundings of 66560 elements average out to less than
# 2^-30 of them; a decay that is short by 0.7·2^-25 a chunk does not.
@pytest.mark.parametrize("dtype,chunk", [(np.float32, 32), (hx.bfloat16, 64)], ids=["f32", "bf16"])
@pytest.mark.parametrize("chunks", [1, 2, 7, 8, 9, 15])
@pytest.mark.parametrize("rest", [0, 1])
def test_a_state_decays_without_drift(device, dtype, chunk, chunks, rest):
    tokens = chunks * chunk + rest
    q, k, v, _, state = operands(dtype, 1, tokens, 260, 260, 16, 16, 22)
    decay = drifting_decays(np.random.default_rng(chunks), 260, chunk)
    v = np.zeros_like(v)
    _, last = run(device, q, k, v, decay, state)
    want = np.exp(decay.astype(np.float64) * tokens)[:, None, None] * state[0]
    assert abs(bias(last[0], want)) <= 2.0**-27


@pytest.mark.parametrize("dtype,chunk", [(np.float32, 32), (hx.bfloat16, 64)], ids=["f32", "bf16"])
@pytest.mark.parametrize("chunks,at", [(8, 7), (8, 6), (8, 0), (9, 8), (9, 7), (16, 14), (11, 3)])
def test_a_token_is_decayed_as_often_as_it_has_to_be(device, dtype, chunk, chunks, at):
    """One token's values, at the end of chunk `at`: what is made good for a
    state's earlier part must not reach them."""
    tokens, t = chunks * chunk, (at + 1) * chunk - 1
    q, k, v, _, _ = operands(dtype, 1, tokens, 260, 260, 16, 16, 23)
    decay = drifting_decays(np.random.default_rng(chunks), 260, chunk)
    v[:, :t], v[:, t + 1:] = np.zeros(1, v.dtype), np.zeros(1, v.dtype)
    _, last = run(device, q, k, v, decay)
    want = (np.exp(decay.astype(np.float64) * (tokens - 1 - t))[:, None, None]
            * as_float64(k)[0, t, :, :, None] * as_float64(v)[0, t, :, None, :])
    assert abs(bias(last[0], want)) <= 2.0**-27


@pytest.mark.parametrize("dtype", [np.float32, hx.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("tokens,heads,dk,dv", [(2048, 300, 32, 32), (512, 300, 32, 32), (2048, 140, 64, 96),
                                                (4096, 2, 64, 64)])
def test_long_memories_keep_the_bits_of_f32(device, dtype, tokens, heads, dk, dv):
    """Heads that remember from four tokens to all, in prompts that are taken
    whole and (the last) cut into parts of a chunk.  Errors in the norm: rounding an
    f32 number errs by 0.2·2^-24 of it.  A state is rounded at most twice a chunk
    and twice a part, at most 256 times: 16·0.2·2^-24; the chunks' own sums and the
    weights (a unit of exp2 each) add 2^-24 each, in all less than 2^-22.  Outputs
    in f32 add as much again at most from sums over a chunk and dk."""
    q, k, v, _, state = operands(dtype, 1, tokens, heads, heads, dk, dv, 24)
    decay = np.log1p(-(2.0 ** -np.linspace(2, 12, heads))).astype(np.float32)
    got, last = run(device, q, k, v, decay, state)
    scale = float(np.float32(dk ** -0.5))
    for h in sorted({0, heads // 4, heads // 2, 3 * heads // 4, heads - 1}):
        want, want_last, _, _ = by_pairs(q[0, :, h], k[0, :, h], v[0, :, h], decay[h], scale, state[0, h])
        assert np.linalg.norm(last[0, h] - want_last) <= 2.0**-22 * np.linalg.norm(want_last), h
        if dtype == np.float32:
            assert np.linalg.norm(got[0, :, h] - want) <= 2.0**-21 * np.linalg.norm(want), h


@pytest.mark.parametrize("dtype", [np.float32, hx.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("tokens,dk", [(1, 16), (3, 16), (1, 48), (1, 100), (1, 200)])
def test_single_tokens_decay_without_drift(device, dtype, tokens, dk):
    """2000 calls on a state in place, with no values: a decay that is a float alone
    is off by up to 2^-25 a token, 2^-14 in the end.  e^g - 1, below 2^-8 here, is
    within two units of its own last place, 2^-30 a token: 2^-19 in 2000."""
    calls, heads = 2000, 40
    q, k, v, _, state = operands(dtype, 1, tokens, heads, heads, dk, 16, 25)
    decay = np.log1p(-(2.0 ** -np.random.default_rng(dk).uniform(8.5, 11, heads))).astype(np.float32)
    off = np.exp(decay.astype(np.float64)) - np.exp(decay.astype(np.float64)).astype(np.float32)
    assert np.abs(off).max() > 2.0**-26  # of a decay near 1: there is something to make good
    v = np.zeros_like(v)
    (vq, _), (vk, _), (vv, _), (vs, read) = (padded(device, x) for x in (q, k, v, state))
    vo, _ = padded(device, v)
    plan = hx.RocmLinearAttentionOps().prepare_linear_attention(device, vq, vk, vv, device.upload(decay), vo,
                                                                state_in=vs, state_out=vs)
    for _ in range(calls):
        plan.dispatch()
    device.synchronize()
    last = read()
    for h in range(heads):
        want = np.exp(decay[h].astype(np.float64) * tokens * calls) * state[0, h]
        assert abs(bias(last[0, h], want)) <= tokens * 2.0**-19, h
