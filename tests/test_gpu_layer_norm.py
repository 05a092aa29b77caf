"""Layer norm and its backward pass against their formulas in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from hephaestus_amd import Layout, StridedView
from layer_reference import EPS32, as_float64, padded, rounded, vector
from training_reference import TYPES, layer_norm, layer_norm_backward, near

pytestmark = pytest.mark.gpu

EPSILON = 1e-5
WIDTHS = [(1, 1), (3, 2), (2, 7), (5, 8), (2, 63), (4, 64), (3, 129), (7, 256), (2, 257), (3, 1000), (2, 1024),
          (2, 1025), (3, 2051), (1, 4096), (5, 4100), (2, 5001), (3, 8193), (2, 16384), (1, 16391), (2, 32771),
          (1, 70001), (300, 96), (1025, 40), (2100, 24)]


def forward(device, x, residual, weight, bias, *, pad=0, offset=0, epsilon=EPSILON, stats=True, keep_h=True):
    vx, _ = padded(device, x, pad, offset)
    vr = None if residual is None else padded(device, residual, pad and pad + 1, offset)[0]
    vy, read_y = padded(device, rounded(np.zeros(x.shape), x.dtype), pad, offset)
    vh, read_h = padded(device, rounded(np.zeros(x.shape), x.dtype), pad, offset)
    mean, rstd = (vector(device, np.full(x.shape[0], -1, np.float32)) for _ in range(2))
    hx.RocmLayerNormOps().layer_norm_into(
        device, vx, vector(device, weight), None if bias is None else vector(device, bias), epsilon, vy, residual=vr,
        residual_out=vh if keep_h else None, mean=mean if stats else None, rstd=rstd if stats else None)
    device.synchronize()
    return {"y": read_y(), "h": read_h() if keep_h else None, "mean": device.download_owned(mean) if stats else None,
            "rstd": device.download_owned(rstd) if stats else None}


def check(got, x, residual, weight, bias, epsilon=EPSILON):
    value, bound = layer_norm(x, residual, weight, bias, epsilon)
    for name, v in got.items():
        if v is not None:
            near(v, value[name], bound[name], name)


def backward(device, dy, h, weight, mean, rstd, past, *, pad=0, offset=0, in_place=None):
    vy, read_dy = padded(device, dy, pad, offset)
    vp, read_past = (None, None) if past is None else padded(device, past, pad, offset)
    vd, read = padded(device, rounded(np.zeros(h.shape), h.dtype), pad, offset)
    if in_place:
        vd, read = (vy, read_dy) if in_place == "grad_out" else (vp, read_past)
    dw, db = (vector(device, np.full(h.shape[1], 7, np.float32)) for _ in range(2))
    hx.RocmLayerNormOps().layer_norm_backward_into(
        device, vy, padded(device, h, pad, offset)[0], vector(device, weight), vector(device, mean),
        vector(device, rstd), vd, residual_grad=vp, grad_weight=dw, grad_bias=db)
    device.synchronize()
    return {"dh": read(), "dw": device.download_owned(dw), "db": device.download_owned(db)}


def operands(t, rows, cols, seed=0, spread=2.0):
    rng = np.random.default_rng(seed)
    x, r, p = (rounded(rng.normal(size=(rows, cols)) * spread + 1, t) for _ in range(3))
    w, b = rounded(rng.uniform(0.5, 1.5, cols), t), rounded(rng.normal(size=cols), t)
    dy = rounded(rng.normal(size=(rows, cols)) * 0.01, t)
    return x, r, w, b, dy, p


def stats_of(h):
    h = as_float64(h)
    return h.mean(1).astype(np.float32), ((h.var(1) + EPSILON)**-0.5).astype(np.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", WIDTHS)
def test_rows_of_every_width(device, dtype, rows, cols):
    x, r, w, b, _, _ = operands(TYPES[dtype], rows, cols, rows * 100003 + cols)
    check(forward(device, x, r, w, b), x, r, w, b)
    check(forward(device, x, None, w, None, stats=False, keep_h=False), x, None, w, None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", WIDTHS)
def test_gradients_of_every_width(device, dtype, rows, cols):
    x, _, w, _, dy, past = operands(TYPES[dtype], rows, cols, rows * 100003 + cols)
    mean, rstd = stats_of(x)
    for p in (past, None):
        got = backward(device, dy, x, w, mean, rstd, p)
        value, bound = layer_norm_backward(dy, x, w, mean, rstd, p)
        for name in got:
            near(got[name], value[name], bound[name], name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,offset", [(1, 0), (3, 1), (8, 3), (5, 7)])
@pytest.mark.parametrize("cols", [37, 512, 4001, 17001, 33000])
def test_strides_and_offsets(device, dtype, pad, offset, cols):
    x, r, w, b, dy, past = operands(TYPES[dtype], 4, cols, cols + pad)
    check(forward(device, x, r, w, b, pad=pad, offset=offset), x, r, w, b)
    mean, rstd = stats_of(x)
    got = backward(device, dy, x, w, mean, rstd, past, pad=pad, offset=offset)
    value, bound = layer_norm_backward(dy, x, w, mean, rstd, past)
    for name in got:
        near(got[name], value[name], bound[name], name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [40, 3000, 20000, 40000])
@pytest.mark.parametrize("in_place", ["grad_out", "residual_grad"])
def test_gradient_in_place(device, dtype, cols, in_place):
    x, _, w, _, dy, past = operands(TYPES[dtype], 37, cols, cols)
    mean, rstd = stats_of(x)
    got = backward(device, dy, x, w, mean, rstd, past, in_place=in_place)
    value, bound = layer_norm_backward(dy, x, w, mean, rstd, past)
    for name in got:
        near(got[name], value[name], bound[name], name)


@pytest.mark.parametrize("cols", [40, 3000, 40000])
@pytest.mark.parametrize("which", ["x", "residual"])
def test_residual_in_place(device, cols, which):
    x, r, w, b, _, _ = operands(hx.bfloat16, 5, cols, cols)
    vx, read_x = padded(device, x)
    vr, read_r = padded(device, r)
    vy, read_y = padded(device, rounded(np.zeros(x.shape), x.dtype))
    hx.RocmLayerNormOps().layer_norm_into(device, vx, vector(device, w), vector(device, b), EPSILON, vy, residual=vr,
                                          residual_out=vx if which == "x" else vr)
    device.synchronize()
    check({"y": read_y(), "h": read_x() if which == "x" else read_r()}, x, r, w, b)


@pytest.mark.parametrize("cols", [40, 3000, 40000])
def test_rows_reversed_and_broadcast(device, cols):
    """A negative row stride, a residual and a gradient that are one row for all."""
    x, r, w, b, dy, _ = operands(np.float32, 5, cols, cols)
    view = StridedView(device.upload(x), Layout.try_new([5, cols], [-cols, 1], 4 * cols))
    one = StridedView(device.upload(r[:1]), Layout.try_new([5, cols], [0, 1]))
    vy, read_y = padded(device, np.zeros_like(x))
    vh, read_h = padded(device, np.zeros_like(x))
    hx.RocmLayerNormOps().layer_norm_into(device, view, vector(device, w), vector(device, b), EPSILON, vy, residual=one,
                                          residual_out=vh)
    device.synchronize()
    all_r = np.repeat(r[:1], 5, 0)
    check({"y": read_y(), "h": read_h()}, x[::-1], all_r, w, b)
    mean, rstd = stats_of(x[::-1])
    same = StridedView(device.upload(dy[:1]), Layout.try_new([5, cols], [0, 1]))
    dw = vector(device, np.zeros(cols, np.float32))
    hx.RocmLayerNormOps().layer_norm_backward_into(device, same, view, vector(device, w), vector(device, mean),
                                                   vector(device, rstd), vy, grad_weight=dw)
    device.synchronize()
    value, bound = layer_norm_backward(np.repeat(dy[:1], 5, 0), x[::-1], w, mean, rstd, None)
    near(read_y(), value["dh"], bound["dh"], "dh")
    near(device.download_owned(dw), value["dw"], bound["dw"], "dw")


@pytest.mark.parametrize("cols", [100, 1000, 20000])
@pytest.mark.parametrize("size", [2.0**-149, 2.0**-140, 2.0**-100, 2.0**-70, 2.0**-40, 2.0**40, 2.0**70, 2.0**120])
def test_sizes_beyond_squares(device, cols, size):
    """Rows whose squares f32 cannot hold, with no epsilon: y does not depend on a
    row's size.  The smallest are whole multiples of the least float."""
    rng = np.random.default_rng(cols)
    x = (rng.integers(-100, 101, (3, cols)) * size).astype(np.float32)
    w, b = np.ones(cols, np.float32), np.zeros(cols, np.float32)
    got = forward(device, x, None, w, b, epsilon=0.0, stats=False, keep_h=False)
    value, bound = layer_norm(x, None, w, b, 0.0)
    near(got["y"], value["y"], bound["y"], "y")


@pytest.mark.parametrize("cols", [1, 100, 1000, 40000])
@pytest.mark.parametrize("value", [0.0, 1.0, -0.1, 1e30, 1e-40])
def test_rows_of_equal_elements(device, cols, value):
    """out is the bias, whatever the rounding of the mean."""
    x = np.full((2, cols), value, np.float32)
    b = np.arange(cols, dtype=np.float32)
    for epsilon in (0.0, EPSILON):
        got = forward(device, x, None, np.ones(cols, np.float32), b, epsilon=epsilon, keep_h=False)
        assert np.array_equal(got["y"], np.repeat(b[None], 2, 0))
        assert np.all(np.abs(got["mean"] - x[:, 0]) <= EPS32 * np.abs(x[:, 0]))
    assert np.all(np.abs(got["rstd"] - EPSILON**-0.5) <= 4 * EPS32 * EPSILON**-0.5) or value == 1e30


def test_values_that_are_no_numbers_stay_in_their_rows(device):
    x, _, w, b, dy, _ = operands(np.float32, 6, 700, 3)
    x[1, 5], x[4, 699] = np.nan, np.inf
    got = forward(device, x, None, w, b, keep_h=False)
    assert np.isnan(got["y"][[1, 4]]).all() and np.isnan(got["mean"][[1, 4]]).sum() >= 1
    rows = [0, 2, 3, 5]
    check({"y": got["y"][rows]}, x[rows], None, w, b)
    back = backward(device, dy, x, w, got["mean"], got["rstd"], None)
    value, bound = layer_norm_backward(dy[rows], x[rows], w, got["mean"][rows], got["rstd"][rows], None)
    near(back["dh"][rows], value["dh"], bound["dh"], "dh")
    assert np.isnan(back["dh"][[1, 4]]).all()


def test_mean_far_from_zero(device):
    """A mean 10^4 times what the elements differ by: the differences are exact, so y
    has the digits that the elements have."""
    rng = np.random.default_rng(5)
    x = (10000 + rng.normal(size=(3, 5000))).astype(np.float32)
    w, b = np.ones(5000, np.float32), np.zeros(5000, np.float32)
    got = forward(device, x, None, w, b, keep_h=False)
    value, _ = layer_norm(x, None, w, b, EPSILON)
    # The mean is rounded to f32 once or twice: 2^-24 of it, 6e-4, in every difference.
    assert np.abs(got["y"] - value["y"]).max() <= 2 * EPS32 * 10000 * value["rstd"].max() * 1.01


def test_no_rows_and_no_columns(device):
    """Sums over no rows are 0."""
    ops, f = hx.RocmLayerNormOps(), np.float32
    empty = StridedView(device.alloc_zeroed(f, 0), Layout.c_contiguous([0, 5]))
    none = device.alloc_zeroed(f, 0)
    dw = vector(device, np.full(5, 3, f))
    five = vector(device, np.ones(5, f))
    ops.layer_norm_into(device, empty, five, None, EPSILON, empty)
    ops.layer_norm_backward_into(device, empty, empty, five, none, none, empty, grad_weight=dw)
    device.synchronize()
    assert np.array_equal(device.download_owned(dw), np.zeros(5, f))
    thin = StridedView(none, Layout.c_contiguous([3, 0]))
    mean = vector(device, np.zeros(3, f))
    ops.layer_norm_into(device, thin, none, None, EPSILON, thin, mean=mean)
    ops.layer_norm_backward_into(device, thin, thin, none, mean, mean, thin, grad_weight=none, grad_bias=none)
    device.synchronize()
    assert np.isnan(device.download_owned(mean)).all()


@pytest.mark.parametrize("cols", [33, 600])
def test_gradient_against_differences(device, cols):
    """Of L = Σ dy·y, by two evaluations in 64 bits an h apart along a direction."""
    x, _, w, b, dy, _ = operands(np.float32, 4, cols, 9)
    got = forward(device, x, None, w, b, keep_h=False)
    back = backward(device, dy, x, w, got["mean"], got["rstd"], None)
    rng = np.random.default_rng(1)
    for name, base in (("dh", x), ("dw", w), ("db", b)):
        way, h = rng.normal(size=base.shape), 1e-4

        def loss(s):
            args = {"dh": x, "dw": w, "db": b}
            args[name] = base.astype(np.float64) + s * way
            xx, ww, bb = args["dh"].astype(np.float64), args["dw"], args["db"]
            u = (xx - xx.mean(1, keepdims=True)) / np.sqrt(xx.var(1, keepdims=True) + EPSILON)
            return (as_float64(dy) * (u * ww + bb)).sum()

        slope = (loss(h) - loss(-h)) / (2 * h)
        size = np.abs(as_float64(back[name]) * way).sum()
        # f32 gradients, and a third derivative's h² of size one.
        assert abs((as_float64(back[name]) * way).sum() - slope) <= 1e-5 * size + 1e-7


def test_runs_repeat_to_the_bit(device):
    x, _, w, _, dy, past = operands(np.float32, 5000, 520, 4)
    mean, rstd = stats_of(x)
    first = backward(device, dy, x, w, mean, rstd, past)
    for _ in range(2):
        again = backward(device, dy, x, w, mean, rstd, past)
        assert all(np.array_equal(first[k], again[k]) for k in first)
