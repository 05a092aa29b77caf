"""How many bits a prompt keeps: linear attention in chunks against closed forms in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from layer_reference import EPS16, EPS32, as_float64, linear_attention
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
