"""The mean that layer norm returns, to the digits that f32 has."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from layer_reference import EPS32, as_float64, rounded
from test_gpu_layer_norm import EPSILON, forward
from training_reference import TYPES

pytestmark = pytest.mark.gpu

# A row each of every kernel: of 16 to 4096 vectors of either type, and longer ones.
COLS = [37, 100, 509, 1003, 2005, 4095, 8191, 16381, 32765, 40007]


def whole(rng, shape, t):
    """Multiples of 2^-7 up to 2 in size: of up to 2^15 of them, and of far more at
    random, every partial sum in f32 is exact, in any order."""
    return rounded(np.clip(np.rint(rng.normal(size=shape) * 64), -256, 256) / 128, t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("has_residual", [False, True])
def test_mean_near_zero_keeps_its_digits(device, dtype, cols, has_residual):
    """The sum is exact and the division rounds once, by EPS32 of the mean, however
    small it is beside the elements.  Twice that is allowed."""
    t, rng = TYPES[dtype], np.random.default_rng(cols)
    x = whole(rng, (50, cols), t)
    r = whole(rng, (50, cols), t) if has_residual else None
    ones, zeros = rounded(np.ones(cols), t), rounded(np.zeros(cols), t)
    got = forward(device, x, r, ones, zeros, keep_h=False)
    h = as_float64(x) + (as_float64(r) if has_residual else 0.0)
    assert np.abs(np.cumsum(h * 128, 1)).max() < 2**24
    mean = h.mean(1)
    assert np.all(np.abs(got["mean"] - mean) <= 2 * EPS32 * np.abs(mean))


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("size", [2.0**-100, 1.0, 2.0**110])
def test_mean_far_from_zero_is_corrected(device, cols, size):
    """A mean 1000 times what the elements differ by: the differences are exact, so
    that what they sum up to corrects the mean, which is rounded once.  Their sum's
    roundings are a thousand times smaller.  Twice the rounding is allowed."""
    rng = np.random.default_rng(cols)
    x = ((1000 + rng.normal(size=(50, cols))).astype(np.float32) * np.float32(size)).astype(np.float32)
    ones, zeros = np.ones(cols, np.float32), np.zeros(cols, np.float32)
    got = forward(device, x, None, ones, zeros, keep_h=False, epsilon=EPSILON * size**2 if size < 2 else EPSILON)
    mean = as_float64(x).mean(1)
    assert np.all(np.abs(got["mean"] - mean) <= 2 * EPS32 * np.abs(mean))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", COLS + [1, 2])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_rows_that_are_not_finite_have_no_mean(device, dtype, cols, value):
    """mean, rstd and out of such a row are NaN, those of its neighbours what they were."""
    t, rng = TYPES[dtype], np.random.default_rng(cols)
    values = as_float64(whole(rng, (3, cols), t))
    values[1, cols // 2] = value
    got = forward(device, rounded(values, t), None, rounded(np.ones(cols), t), rounded(np.zeros(cols), t), keep_h=False)
    for name in ("mean", "rstd"):
        assert np.isnan(got[name][1]) and np.isfinite(got[name][[0, 2]]).all()
    y = as_float64(got["y"])
    assert np.isnan(y[1]).all() and np.isfinite(y[[0, 2]]).all()
