"""States that are infinite."""
from __future__ import annotations

import numpy as np
import pytest

from layer_reference import as_float64, rounded
from test_gpu_gated_recurrence import backward, forward
from training_reference import TYPES

pytestmark = pytest.mark.gpu

SIZES = [(2, 1, 70), (64, 1, 130), (2, 2, 70), (2, 20, 70), (3, 32, 65)]  # up to one wave's tokens
LONGER = [(1, 120, 70), (200, 130, 64), (1, 700, 70)]  # tiles of 64 and 128 tokens, parts


def gates(tokens, channels, t):
    """From nearly shut (f = 1/8) to nearly open, such that the factors of all tokens
    together are above 2^-126."""
    least = max(2.0**-3, 2.0**(-120 / tokens))
    f = np.linspace(least, 0.999, channels)
    return rounded(np.log(f / (1 - f)) + 0.01, t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,tokens,channels", SIZES)
def test_an_infinite_state_stays_one(device, dtype, batch, tokens, channels):
    """f·h and h - (1 - f)·h both are infinite, whichever way a factor is applied; the
    gradient of the last state alike."""
    t = TYPES[dtype]
    gate = np.broadcast_to(gates(tokens, channels, t), (batch, tokens, channels)).copy()
    x = rounded(np.random.default_rng(1).normal(size=gate.shape), t)
    first = np.full((batch, channels), np.inf, np.float32)
    first[:, ::2] = -np.inf
    got = forward(device, gate, x, first)
    want = np.broadcast_to(first[:, None], gate.shape)
    assert np.array_equal(as_float64(got["h"]), want) and np.array_equal(got["last"], first)
    dy = rounded(np.zeros(gate.shape), t)
    back = backward(device, gate, x, rounded(np.zeros(gate.shape), t), dy, None, first)
    assert np.array_equal(as_float64(back["dx"]), want) and np.array_equal(back["dfirst"], first)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,tokens,channels", LONGER)
def test_an_infinite_state_of_many_tokens_stays_in_its_channel(device, dtype, batch, tokens, channels):
    t = TYPES[dtype]
    gate = np.broadcast_to(gates(tokens, channels, t), (batch, tokens, channels)).copy()
    x = rounded(np.random.default_rng(1).normal(size=gate.shape), t)
    first = np.zeros((batch, channels), np.float32)
    first[:, ::2] = -np.inf
    got = forward(device, gate, x, first)
    for out in (as_float64(got["h"])[..., ::2], got["last"][:, ::2]):
        assert not np.isfinite(out).any() and not (out > 0).any()
    assert np.isfinite(as_float64(got["h"])[..., 1::2]).all() and np.isfinite(got["last"][:, 1::2]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [20, 700])
def test_an_infinite_input_stays_in_its_channel(device, dtype, tokens):
    """It reaches the later outputs as an infinity or a NaN, and no others; the outputs of
    the token itself are infinite."""
    t = TYPES[dtype]
    gate = np.broadcast_to(gates(tokens, 70, t), (1, tokens, 70)).copy()
    values = np.random.default_rng(1).normal(size=gate.shape)
    at = 2 * tokens // 3
    values[0, at, ::2] = np.inf
    got = as_float64(forward(device, gate, rounded(values, t), None)["h"])
    assert np.isfinite(got[0, :at]).all() and np.isfinite(got[0, :, 1::2]).all()
    assert np.all(got[0, at, ::2] == np.inf) and not np.isfinite(got[0, at:, ::2]).any()
