"""Operands of linear attention that are no numbers: what they reach, and what they must not."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from layer_reference import as_float64, linear_attention, rounded
from test_gpu_linear_attention import TYPES, operands, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 5, 20, 64, 70, 1500])
def test_a_decay_that_is_no_number_spoils_its_head_only(device, dtype, tokens):
    """In single tokens, within a chunk, over chunks and in a prompt that is cut."""
    q, k, v, decay, state = operands(TYPES[dtype], 1, tokens, 3, 3, 32, 32, 31)
    decay[1] = np.nan
    for first in (state, None):
        got, last = run(device, q, k, v, decay, first)
        got = as_float64(got)
        assert np.isnan(got[:, :, 1]).all() and np.isnan(last[:, 1]).all()
        assert np.isfinite(np.delete(got, 1, 2)).all() and np.isfinite(np.delete(last, 1, 1)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 5, 70, 4100])
def test_a_sequence_of_no_tokens_keeps_any_state(device, dtype, tokens):
    """To the bit, infinities, NaN and negative zeros too; beside it a sequence
    that ends where a part of a cut prompt does."""
    q, k, v, decay, state = operands(TYPES[dtype], 2, tokens, 1, 1, 16, 16, 32)
    state[0, 0, 3, :4] = np.inf, -np.inf, np.nan, -0.0
    state[0, 0, 9, 5:7] = -0.0, 1e-40
    got, last = run(device, q, k, v, decay, state, [0, tokens])
    assert np.array_equal(last[0].view(np.uint32), state[0].view(np.uint32))
    assert not as_float64(got)[0].any() and np.isfinite(last[1]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 6, 70, 700])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("where", ["q", "k", "v", "state"])
def test_what_is_not_finite_reaches_what_the_formula_says(device, dtype, tokens, value, where):
    """Which of infinity and NaN it is depends on the order of the sums."""
    q, k, v, decay, state = operands(TYPES[dtype], 1, tokens, 2, 1, 32, 32, 33)
    state = state.copy()
    t = tokens // 2
    bad = rounded(np.array([value]), TYPES[dtype])[0]
    if where == "state":
        state[0, 1, 7, 3] = value
    else:
        {"q": q, "k": k, "v": v}[where][0, t, 0, 7] = bad
    got, last = run(device, q, k, v, decay, state)
    with np.errstate(invalid="ignore"):
        want, want_last, _, _ = linear_attention(q, k, v, decay, 32 ** -0.5, state)
    assert np.array_equal(np.isfinite(as_float64(got)), np.isfinite(want))
    assert np.array_equal(np.isfinite(last), np.isfinite(want_last))
