"""Losses of rows that are nearly sure of their target: small numbers beside logits in
the hundreds."""
from __future__ import annotations

import numpy as np
import pytest

from layer_reference import EPS32, rounded
from test_gpu_cross_entropy import forward
from training_reference import TYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,width", [(5, 300, 8), (40, 5000, 8), (300, 1000, 24), (2100, 700, 8), (16, 100, 4096)])
def test_loss_keeps_the_digits_of_the_sum(device, dtype, rows, vocab, width):
    """Logits that are exact in any order of summation: 300 of the target, 288 and 290
    of two words more, 0 of all others.  The loss is log(1 + e^-12 + e^-10) = 5.2e-5;
    half a step of f32 at 300 is 1.5e-5.  The sum of exponentials is rounded when each of
    the two is added and once more where tiles meet, by EPS32 each, and its logarithm
    once."""
    t, rng = TYPES[dtype], np.random.default_rng(rows)
    words = np.array([rng.choice(vocab, 3, replace=False) for _ in range(8)])
    x, w = np.zeros((rows, width)), np.zeros((vocab, width))
    kind = np.arange(rows) % 8
    x[np.arange(rows), kind] = 1
    for j in range(8):
        w[words[j], j] = [300, 288, 290]
    targets = words[kind, 0].astype(np.uint32)
    got = forward(device, rounded(x, t), rounded(w, t), targets)
    want = np.log1p(np.exp(-12.0) + np.exp(-10.0))
    assert np.abs(got["loss"] - want).max() <= 4 * EPS32
    assert np.abs(got["lse"] - (300 + want)).max() <= 2 * EPS32 * 300
    # The second word's loss is 12 more: its rounding is that of 12.
    got = forward(device, rounded(x, t), rounded(w, t), words[kind, 1].astype(np.uint32), lse=False)
    assert np.abs(got["loss"] - (12 + want)).max() <= 4 * EPS32 + 2 * EPS32 * 12
