"""The example model: it runs in both types, its gradients are those of the whole
model's formula in 64 bits, and a prompt of any lengths gives the same gradients
for what lies within them."""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import pytest

import hephaestus_amd as hx

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
import recurrent_language_model as example  # noqa: E402

pytestmark = pytest.mark.gpu

SIZES = {"vocab": 50, "width": 24, "batch": 3, "tokens": 40}


def loss_of(parameters, text, lengths, width):
    """The mean loss in 64 bits."""
    embedding, weight, bias, head = parameters
    words, following = text[:, :-1], text[:, 1:]
    x = embedding[words]
    d = x - x.mean(-1, keepdims=True)
    y = d / np.sqrt((d * d).mean(-1, keepdims=True) + example.EPSILON) * weight + bias
    f, u = 1 / (1 + np.exp(-y[..., :width])), y[..., width:]
    state, total = np.zeros((len(text), width)), 0.0
    for t in range(words.shape[1]):
        state = f[:, t] * state + (1 - f[:, t]) * u[:, t]
        logits = state @ head.T
        top = logits.max(1)
        lse = top + np.log(np.exp(logits - top[:, None]).sum(1))
        total += ((lse - logits[np.arange(len(text)), following[:, t]]) * (t < lengths)).sum()
    return total / lengths.sum()


def test_gradients_against_differences(device):
    model = example.Model(device, **SIZES)
    text, lengths = example.text_of(3, 40, 50)
    lengths[0] = 7
    loss, gradients = model.step(text, lengths)
    names = ["embedding", "norm_weight", "norm_bias", "head"]
    base = [getattr(model, n).astype(np.float64) for n in names]
    # f32 along a row's sums and 40 tokens: some hundred roundings of 2^-24.
    assert abs(loss - loss_of(base, text, lengths, 24)) <= 1e-5 * loss
    rng = np.random.default_rng(0)
    for i, name in enumerate(names):
        way, h = rng.normal(size=base[i].shape), 1e-4
        slope = 0.0
        for sign in (1, -1):
            moved = list(base)
            moved[i] = base[i] + sign * h * way
            slope += sign * loss_of(moved, text, lengths, 24) / (2 * h)
        got = gradients[name].astype(np.float64)
        # Hundreds of roundings of 2^-24 a term, and h² of a third derivative of size one.
        assert abs((got * way).sum() - slope) <= 5e-5 * np.abs(got * way).sum() + 1e-7, name


def test_bfloat16_runs_near_f32(device):
    text, lengths = example.text_of(3, 40, 50)
    (loss, gradients), (loss16, gradients16) = (
        example.Model(device, dtype=t, **SIZES).step(text, lengths) for t in (np.float32, hx.bfloat16))
    # Parameters, activations and gradients are rounded by up to 2^-8 each, some ten
    # times between a parameter and its gradient.
    assert abs(loss - loss16) <= 10 * 2.0**-8 * loss
    for name in gradients:
        off = np.linalg.norm(gradients16[name] - gradients[name]) / np.linalg.norm(gradients[name])
        assert off <= 10 * 2.0**-8, name


def test_what_lies_past_a_length_does_not_count(device):
    model = example.Model(device, **SIZES)
    text, lengths = example.text_of(3, 40, 50)
    first = model.step(text, lengths)
    for b, n in enumerate(lengths):
        text[b, n + 1:] = (text[b, n + 1:] + 11) % 50
    again = model.step(text, lengths)
    assert first[0] == again[0]
    for name in first[1]:
        assert np.array_equal(first[1][name], again[1][name]), name


def test_steps_run(device):
    model = example.Model(device, dtype=hx.bfloat16, **SIZES)
    for seed in range(3):
        loss, gradients = model.step(*example.text_of(3, 40, 50, seed))
        model.update(gradients, rate=0.5)
        assert np.isfinite(loss)
    assert all(np.isfinite(getattr(model, n)).all() for n in ("embedding", "norm_weight", "norm_bias", "head"))
