"""RMS norm of rows whose squares are too small for f32, where epsilon does not
outweigh them."""
from __future__ import annotations

import numpy as np
import pytest

from layer_reference import as_float64, padded, rounded
from test_gpu_norm_quantize import TYPES, check, run

import hephaestus_amd as hx

pytestmark = pytest.mark.gpu

# Widths of every form: several rows a wave, a wave, blocks, two and four vectors a
# thread, rows that are read twice; a whole number of vectors and not.
COLS = [24, 61, 200, 450, 1000, 2048, 3001, 5001, 12000, 16391, 40000]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("epsilon", [0.0, 1e-44, 1e-36])
def test_rows_down_to_the_least_float(device, dtype, cols, epsilon):
    t = TYPES[dtype]
    rng = np.random.default_rng(cols)
    sizes = [1.0, 1e-15, 1e-17, 1e-18, 3e-19, 1e-20, 1e-21, 1e-23, 1e-30, 1e-37, 1e-42, 0.0, 1e10]
    x = rounded(rng.normal(size=(len(sizes), cols)) * np.array(sizes)[:, None], t)
    w = rounded(rng.uniform(0.5, 1.5, cols), t)
    got = run(device, x, None, w, keep_h=False, epsilon=epsilon)
    live = as_float64(x).any(axis=1)  # 1e-42 is below the least bf16
    assert live[:10].all() and not live[11]
    check(x[live], None, w, (None, got[1][live], got[2][live]), float(np.float32(epsilon)))
    assert np.all(got[2][live] > 0) and not got[1][~live].any() and not got[2][~live].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", COLS)
def test_one_element_of_a_tiny_row(device, dtype, cols):
    """All else is zero: y is that element's sign, √cols and its weight."""
    t = TYPES[dtype]
    x = np.zeros((4, cols), np.float32)
    x[np.arange(4), [0, cols // 2, cols - 1, 3]] = 1e-25, -1e-30, 2e-38, -1e-22
    w = rounded(np.full(cols, 2.0**-70), t)
    _, q, scales = run(device, rounded(x, t), None, w, keep_h=False, epsilon=0.0)
    assert np.count_nonzero(q) == 4
    assert [int(q[i, c]) for i, c in enumerate([0, cols // 2, cols - 1, 3])] == [127, -127, 127, -127]
    want = np.sqrt(cols) * 2.0**-70 / 127
    assert np.all(np.abs(scales - want) <= want * 40 * 2.0**-24)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [61, 2048, 5001, 40000])
def test_tiny_rows_with_the_residual_in_place(device, dtype, cols):
    """Among ordinary rows; h lies where x was, and is read until it is written."""
    t = TYPES[dtype]
    rng = np.random.default_rng(cols)
    sizes = np.array([1e-25, 1.0, 1e-25, 1e-25, 1e-38, 5.0])[:, None]
    x, r = (rounded(rng.normal(size=(6, cols)) * sizes, t) for _ in range(2))
    w = rounded(rng.uniform(0.5, 2, cols), t)
    vx, read_x = padded(device, x, 3)
    vr, _ = padded(device, r, 5)
    vq, read_q = padded(device, np.zeros((6, cols), np.int8))
    scales = device.alloc_zeroed(np.float32, 6)
    hx.RocmNormOps().rms_norm_quantize_into(device, vx, device.upload(w), 0.0, vq, scales, residual=vr,
                                            residual_out=vx)
    device.synchronize()
    check(x, r, w, (read_x(), read_q(), device.download_owned(scales)), 0.0)


@pytest.mark.parametrize("cols", [61, 2048, 40000])
def test_weights_that_are_no_numbers_in_tiny_rows(device, cols):
    x = np.full((2, cols), 1e-25, np.float32)
    for bad in (np.nan, np.inf):
        w = np.ones(cols, np.float32)
        w[cols - 3] = bad
        _, q, scales = run(device, x, None, w, keep_h=False, epsilon=0.0)
        assert np.isnan(scales).all() and not q.any()
