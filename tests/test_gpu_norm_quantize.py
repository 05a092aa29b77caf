"""RMS norm with the residual's addition and an 8-bit output against its
formula in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from layer_reference import EPS16, EPS32, as_float64, norm_quantize, padded, rounded, vector

pytestmark = pytest.mark.gpu

TYPES = {"f32": np.float32, "bf16": hx.bfloat16}
EPSILON = 1e-5


def run(device, x, residual, weight, *, keep_h=True, pad=0, offset=0, epsilon=EPSILON, prepared=False):
    vx, _ = padded(device, x, pad, offset)
    vr = None if residual is None else padded(device, residual, pad and pad + 1, offset)[0]
    vq, read_q = padded(device, np.full(x.shape, 55, np.int8), pad, offset)
    vh, read_h = padded(device, rounded(np.zeros(x.shape), x.dtype), pad, offset)
    scales = vector(device, np.full(x.shape[0], -1, np.float32))
    args = (device, vx, vector(device, weight), epsilon, vq, scales)
    more = {"residual": vr, "residual_out": vh if keep_h else None}
    if prepared:
        plan = hx.RocmNormOps().prepare_rms_norm_quantize(*args, **more)
        plan.dispatch()
        plan.dispatch()
    else:
        hx.RocmNormOps().rms_norm_quantize_into(*args, **more)
    device.synchronize()
    return read_h() if keep_h else None, read_q(), device.download_owned(scales)


def check(x, residual, weight, got, epsilon=EPSILON):
    h, steps, s = norm_quantize(x, residual, weight, epsilon)
    got_h, q, scales = got
    cols = x.shape[1]
    if got_h is not None:
        terms = np.abs(as_float64(x)) + (0 if residual is None else np.abs(as_float64(residual)))
        assert np.all(np.abs(as_float64(got_h) - h) <= terms * EPS32 + np.abs(h) * (EPS16 if x.dtype == hx.bfloat16 else 0))
    # A sum of `cols` squares folded over 64 lanes or more, a root, a quotient.
    assert np.all(np.abs(scales - s) <= s * (cols / 64 + 40) * EPS32)
    # Half a step, and the roundings of h, h·w, 127 / top and the product.
    assert np.all(np.abs(q - steps) <= 0.5 + 127 * 8 * EPS32)
    assert np.abs(q.astype(int)).max(initial=0) <= 127


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [
    (1, 1), (3, 2), (1, 7), (5, 8), (2, 63), (4, 64), (3, 255), (7, 256), (2, 257), (3, 1000), (2, 1024), (2, 1025),
    (3, 2048), (2, 2051), (1, 4096), (5, 4100), (2, 5001), (3, 8192), (2, 8193), (1, 16384), (2, 16391), (1, 32768),
    (2, 32771), (1, 70001), (300, 96), (1025, 40)])
def test_rows_of_every_width(device, dtype, rows, cols):
    rng = np.random.default_rng(rows * 100003 + cols)
    t = TYPES[dtype]
    x, r = (rounded(rng.normal(size=(rows, cols)) * 2, t) for _ in range(2))
    w = rounded(rng.uniform(0.5, 1.5, cols), t)
    check(x, r, w, run(device, x, r, w))
    check(x, None, w, run(device, x, None, w, keep_h=False))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,offset", [(1, 0), (3, 1), (8, 3), (16, 16), (5, 7)])
@pytest.mark.parametrize("cols", [37, 512, 3000, 9000])
def test_strides_and_offsets(device, dtype, pad, offset, cols):
    rng = np.random.default_rng(cols + pad)
    t = TYPES[dtype]
    x, r = (rounded(rng.normal(size=(4, cols)), t) for _ in range(2))
    w = rounded(rng.normal(size=cols), t)
    check(x, r, w, run(device, x, r, w, pad=pad, offset=offset, prepared=True))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [40, 3000, 40000])
def test_rows_reversed_and_broadcast(device, dtype, cols):
    """A negative row stride, and a residual that is one row for all."""
    rng = np.random.default_rng(cols)
    t = TYPES[dtype]
    x, r = rounded(rng.normal(size=(5, cols)), t), rounded(rng.normal(size=(1, cols)), t)
    w = rounded(rng.uniform(0.5, 2, cols), t)
    buffer, rb = device.upload(x), device.upload(r)
    q = device.alloc_zeroed(np.int8, 5 * cols)
    scales = device.alloc_zeroed(np.float32, 5)
    hx.RocmNormOps().rms_norm_quantize_into(
        device, hx.StridedView(buffer, hx.Layout.try_new([5, cols], [-cols, 1], 4 * cols)), device.upload(w), EPSILON,
        hx.StridedView(q, hx.Layout.c_contiguous([5, cols])), scales,
        residual=hx.StridedView(rb, hx.Layout.try_new([5, cols], [0, 1])))
    device.synchronize()
    check(x[::-1], np.repeat(r, 5, 0), w,
          (None, device.download_owned(q).reshape(5, cols), device.download_owned(scales)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [33, 4096, 33000])
@pytest.mark.parametrize("place", ["x", "residual"])
def test_residual_in_place(device, dtype, cols, place):
    rng = np.random.default_rng(cols)
    t = TYPES[dtype]
    x, r = (rounded(rng.normal(size=(6, cols)), t) for _ in range(2))
    w = rounded(rng.uniform(0.5, 2, cols), t)
    vx, read_x = padded(device, x, 3)
    vr, read_r = padded(device, r, 3)
    vq, read_q = padded(device, np.zeros((6, cols), np.int8))
    scales = device.alloc_zeroed(np.float32, 6)
    hx.RocmNormOps().rms_norm_quantize_into(device, vx, device.upload(w), EPSILON, vq, scales, residual=vr,
                                            residual_out=vx if place == "x" else vr)
    device.synchronize()
    check(x, r, w, ((read_x if place == "x" else read_r)(), read_q(), device.download_owned(scales)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [24, 4096, 40000])
def test_rows_that_cannot_be_scaled(device, dtype, cols):
    t = TYPES[dtype]
    x = np.random.default_rng(1).normal(size=(7, cols)).astype(np.float32)
    x[0] = 0
    x[1, cols // 2] = np.nan
    x[2, cols - 1] = np.inf
    x[3, 0] = -np.inf
    x[4] = 3e38          # the squares leave f32
    x[5] *= 1e-30        # tiny, but the norm brings it back
    x[6] = 0
    x[6, 5] = 2          # one element
    x = rounded(x, t)
    for epsilon in (0.0, 1e-5):
        _, q, scales = run(device, x, None, rounded(np.ones(cols), t), keep_h=False, epsilon=epsilon)
        assert scales[0] == 0 and not q[0].any()
        assert np.isnan(scales[1:5]).all() and not q[1:5].any()
        live = [6] if epsilon == 0 else [5, 6]  # squares of 1e-30 vanish in f32
        check(x[live], None, rounded(np.ones(cols), t), (None, q[live], scales[live]), epsilon)
        assert q[6, 5] == 127 and np.count_nonzero(q[6]) == 1


@pytest.mark.parametrize("dtype", TYPES)
def test_weight_not_a_number(device, dtype):
    t = TYPES[dtype]
    x = rounded(np.random.default_rng(2).normal(size=(2, 300)), t)
    for bad in (np.nan, np.inf):
        w = np.ones(300, np.float32)
        w[77] = bad
        _, q, scales = run(device, x, None, rounded(w, t), keep_h=False)
        assert np.isnan(scales).all() and not q.any()


def test_tiny_weights_keep_all_steps(device):
    """Rows whose scale is near the least f32: 127 / max|h·w| would overflow."""
    x = np.random.default_rng(3).normal(size=(3, 500)).astype(np.float32)
    w = np.full(500, 2.0**-124, np.float32)
    h, steps, _ = norm_quantize(x, None, w, EPSILON)
    _, q, scales = run(device, x, None, w, keep_h=False)
    assert np.all(np.abs(q - steps) <= 0.51)  # h·w keeps at least 20 bits
    assert np.all(scales > 0)


def test_no_rows_and_no_columns(device):
    for rows, cols in ((0, 64), (3, 0)):
        _, q, scales = run(device, np.zeros((rows, cols), np.float32), None, np.ones(cols, np.float32), keep_h=False)
        assert q.shape == (rows, cols) and not scales.any()


@pytest.mark.parametrize("residual", [False, True])
def test_more_rows_than_a_launch_takes(device, residual):
    """Sixteen rows a block and at most 2^21 blocks a launch."""
    rows = 2**25 + 21
    x = ((np.arange(rows) * 7) % 97 - 48).astype(np.float32)[:, None]
    r = np.flip(x, 0).copy() if residual else None
    w = np.full(1, 1.25, np.float32)
    check(x, r, w, run(device, x, r, w, keep_h=residual))
