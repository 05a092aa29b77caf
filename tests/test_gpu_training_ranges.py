"""The ends of the ranges that include/hx.h states for gradients."""
from __future__ import annotations

import numpy as np
import pytest

from layer_reference import as_float64, rounded
from test_gpu_cross_entropy import backward as loss_backward, lse_of, operands as loss_operands
from test_gpu_layer_norm import backward as norm_backward, forward as norm_forward
from training_reference import TYPES, cross_entropy_backward, layer_norm_backward, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [60, 600])
def test_rows_of_very_different_gradients(device, dtype, rows):
    """Rows 2^-90 of the largest keep their own digits in grad_x."""
    x, w, targets, grad = loss_operands(TYPES[dtype], rows, 130, 50, 9)
    grad[::2] *= np.float32(2.0**-90)
    lse = lse_of(x, w)
    got = loss_backward(device, x, w, targets, lse, grad)
    value, bound = cross_entropy_backward(x, w, targets, lse, grad)
    for name in got:
        near(got[name], value[name], bound[name], name)


@pytest.mark.parametrize("cols", [100, 3000, 40000])
@pytest.mark.parametrize("size", [2.0**-120, 2.0**-60, 2.0**60, 2.0**118])
def test_gradients_of_rows_of_any_size(device, cols, size):
    """rstd is within f32: so are the gradients' differences from the mean."""
    rng = np.random.default_rng(cols)
    x = (rng.integers(-100, 101, (4, cols)) / 64 * size).astype(np.float32)
    w = rng.uniform(0.5, 1.5, cols).astype(np.float32)
    dy = (rng.normal(size=(4, cols)) * min(1.0, size)).astype(np.float32)
    got = norm_forward(device, x, None, w, np.zeros(cols, np.float32), epsilon=0.0, keep_h=False)
    assert np.isfinite(got["rstd"]).all()
    back = norm_backward(device, dy, x, w, got["mean"], got["rstd"], None)
    value, bound = layer_norm_backward(dy, x, w, got["mean"], got["rstd"], None)
    for name in back:
        near(back[name], value[name], bound[name], name)


@pytest.mark.parametrize("cols", [100, 3000, 40000])
def test_rstd_past_f32_is_infinite(device, cols):
    """out is what it should be all the same."""
    rng = np.random.default_rng(cols)
    x = (rng.integers(-3, 4, (3, cols)) * 2.0**-145).astype(np.float32)
    x[1] *= np.float32(2.0**80)
    got = norm_forward(device, x, None, np.ones(cols, np.float32), np.zeros(cols, np.float32), epsilon=0.0, keep_h=False)
    assert np.isinf(got["rstd"][[0, 2]]).all() and np.isfinite(got["rstd"][1])
    h = as_float64(x)
    want = (h - h.mean(1, keepdims=True)) / h.std(1, keepdims=True)
    assert np.abs(got["y"] - want).max() <= 1e-5 * np.abs(want).max()
