"""Gradients of losses whose vocabulary is taken in pieces, with grad_x in parts of each
piece's words and without."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_cross_entropy import backward, forward, operands
from training_reference import TYPES, cross_entropy_backward, near

pytestmark = pytest.mark.gpu

# (type, rows, words, width) by whether grad_x of every piece is cut into parts.
PARTS = [("bf16", 600, 300000, 64), ("f32", 300, 300000, 64)]
WHOLE = [("bf16", 70000, 4500, 8), ("f32", 70000, 2000, 40)]


@pytest.mark.parametrize("dtype,rows,vocab,width", PARTS + WHOLE)
def test_pieces(device, dtype, rows, vocab, width):
    x, w, targets, grad = operands(TYPES[dtype], rows, vocab, width, 13)
    lse = forward(device, x, w, targets)["lse"]
    got = backward(device, x, w, targets, lse, grad)
    rng = np.random.default_rng(2)
    part = np.sort(rng.choice(rows, 40, replace=False))
    value, bound = cross_entropy_backward(x[part], w, targets[part], lse[part], grad[part])
    near(got["dx"][part], value["dx"], bound["dx"], "dx")
    # Some words of every piece: those first and last, and those that are targets.  All
    # other targets are one word more, whose gradient is not looked at.
    words = np.unique(np.concatenate([[0, 1, vocab // 2 - 1, vocab // 2, vocab - 2, vocab - 1], rng.choice(vocab, 20),
                                      targets[targets < vocab][:20]])).astype(np.int64)
    place = np.full(vocab, len(words))
    place[words] = np.arange(len(words))
    has = targets < vocab
    moved = np.where(has, place[np.where(has, targets, 0)], targets).astype(np.uint32)
    value, bound = cross_entropy_backward(x, np.concatenate([w[words], w[:1]]), moved, lse, grad)
    near(got["dw"][words], value["dw"][:-1], bound["dw"][:-1], "dw")
