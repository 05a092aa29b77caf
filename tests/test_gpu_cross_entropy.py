"""Softmax cross entropy over a vocabulary and its backward pass against their
formulas in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from hephaestus_amd import NO_TARGET, Layout, StridedView
from layer_reference import as_float64, padded, rounded, vector
from training_reference import TYPES, cross_entropy, cross_entropy_backward, near

pytestmark = pytest.mark.gpu

SIZES = [(1, 1, 1), (1, 2, 3), (3, 5, 7), (1, 1000, 64), (16, 333, 100), (17, 64, 63), (31, 65, 65), (32, 700, 256),
         (33, 129, 130), (64, 64, 64), (65, 1025, 33), (100, 77, 513), (129, 127, 96), (200, 600, 200), (257, 260, 70),
         (500, 33, 2), (40, 20000, 16), (1030, 2050, 40), (2100, 5300, 24)]


def operands(t, rows, vocab, width, seed=0, left_out=0.2):
    rng = np.random.default_rng(seed)
    x = rounded(rng.normal(size=(rows, width)), t)
    w = rounded(rng.normal(size=(vocab, width)) * 2 / np.sqrt(width), t)
    targets = rng.integers(0, vocab, rows).astype(np.uint32)
    targets[rng.random(rows) < left_out] = NO_TARGET
    return x, w, targets, rng.uniform(0.5, 1.5, rows).astype(np.float32) / max(1, rows)


def forward(device, x, w, targets, *, lse=True, **place):
    loss, out = (vector(device, np.full(x.shape[0], 7, np.float32)) for _ in range(2))
    hx.RocmLossOps().linear_cross_entropy_into(device, padded(device, x, **place)[0], padded(device, w, **place)[0],
                                               vector(device, targets), loss, out if lse else None)
    device.synchronize()
    return {"loss": device.download_owned(loss), **({"lse": device.download_owned(out)} if lse else {})}


def backward(device, x, w, targets, lse, grad, names=("dx", "dw"), **place):
    views = {"dx": padded(device, rounded(np.full(x.shape, 7.0), x.dtype), **place),
             "dw": padded(device, rounded(np.full(w.shape, 7.0), x.dtype), **place)}
    hx.RocmLossOps().linear_cross_entropy_backward_into(
        device, padded(device, x, **place)[0], padded(device, w, **place)[0], vector(device, targets),
        vector(device, lse), vector(device, grad), grad_x=views["dx"][0] if "dx" in names else None,
        grad_weight=views["dw"][0] if "dw" in names else None)
    device.synchronize()
    return {name: views[name][1]() for name in names}


def check(got, expected):
    value, bound = expected
    for name in got:
        near(got[name], value[name], bound[name], name)


def lse_of(x, w):
    logits = as_float64(x) @ as_float64(w).T
    top = logits.max(1)
    return (top + np.log(np.exp(logits - top[:, None]).sum(1))).astype(np.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,width", SIZES)
def test_sizes(device, dtype, rows, vocab, width):
    x, w, targets, grad = operands(TYPES[dtype], rows, vocab, width, rows + vocab + width)
    check(forward(device, x, w, targets), cross_entropy(x, w, targets))
    lse = lse_of(x, w)
    check(backward(device, x, w, targets, lse, grad), cross_entropy_backward(x, w, targets, lse, grad))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("names", [("dx",), ("dw",)])
def test_one_gradient(device, dtype, names):
    x, w, targets, grad = operands(TYPES[dtype], 70, 300, 90, 1)
    lse = lse_of(x, w)
    check(backward(device, x, w, targets, lse, grad, names), cross_entropy_backward(x, w, targets, lse, grad))
    check(forward(device, x, w, targets, lse=False), cross_entropy(x, w, targets))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("place", [{"strides_pad": 1}, {"strides_pad": 2, "offset": 1}, {"offset": 3},
                                   {"strides_pad": 8, "offset": 8}])
@pytest.mark.parametrize("rows,vocab,width", [(5, 70, 33), (130, 200, 64), (300, 260, 130)])
def test_strides(device, dtype, place, rows, vocab, width):
    x, w, targets, grad = operands(TYPES[dtype], rows, vocab, width, 4)
    check(forward(device, x, w, targets, **place), cross_entropy(x, w, targets))
    lse = lse_of(x, w)
    check(backward(device, x, w, targets, lse, grad, **place), cross_entropy_backward(x, w, targets, lse, grad))


def test_rows_reversed_and_broadcast(device):
    """A negative stride of the rows, and one word's weights for a whole vocabulary:
    its gradients are each a row's own."""
    x, w, targets, grad = operands(np.float32, 9, 1, 40, 4, left_out=0)
    targets = np.arange(9, dtype=np.uint32)
    flipped = StridedView(device.upload(x), Layout.try_new([9, 40], [-40, 1], 8 * 40))
    same = StridedView(device.upload(w), Layout.try_new([12, 40], [0, 1]))
    loss, lse = (vector(device, np.zeros(9, np.float32)) for _ in range(2))
    ops, at = hx.RocmLossOps(), vector(device, targets)
    ops.linear_cross_entropy_into(device, flipped, same, at, loss, lse)
    vx, read_x = padded(device, np.zeros_like(x))
    vw, read_w = padded(device, np.zeros((12, 40), np.float32))
    ops.linear_cross_entropy_backward_into(device, flipped, same, at, lse, vector(device, grad), vx, vw)
    device.synchronize()
    all_w = np.repeat(w, 12, 0)
    check({"loss": device.download_owned(loss), "lse": device.download_owned(lse)}, cross_entropy(x[::-1], all_w, targets))
    check({"dx": read_x(), "dw": read_w()},
          cross_entropy_backward(x[::-1], all_w, targets, device.download_owned(lse), grad))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 200])
def test_rows_left_out(device, dtype, rows):
    """Whatever a row without a target holds, it adds nothing; any target from the
    vocabulary on leaves its row out, and all rows may be."""
    x, w, targets, grad = operands(TYPES[dtype], rows, 150, 70, 6)
    lse = lse_of(x, w)
    targets[::3] = [150, NO_TARGET, 151][rows % 3]
    clean = x.copy()
    nan = rounded(np.array([np.nan]), x.dtype)[0]
    x[::3], grad[::3], lse[::3] = nan, np.nan, np.inf
    clean[::3] = rounded(np.array([0.0]), x.dtype)[0]
    got = forward(device, x, w, targets)
    assert not got["loss"][::3].any()
    rest = targets < 150
    value, bound = cross_entropy(clean, w, targets)
    near(got["loss"][rest], value["loss"][rest], bound["loss"][rest], "loss")
    back = backward(device, x, w, targets, lse, grad)
    clean_lse, clean_grad = np.where(np.isfinite(lse), lse, 0), np.where(np.isfinite(grad), grad, 0)
    check(back, cross_entropy_backward(clean, w, targets, clean_lse.astype(np.float32), clean_grad.astype(np.float32)))
    assert not as_float64(back["dx"][::3]).any()
    none = np.full(rows, NO_TARGET, np.uint32)
    back = backward(device, x, w, none, lse, grad)
    assert not as_float64(back["dx"]).any() and not as_float64(back["dw"]).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [30.0, 300.0])
def test_sharp_distributions(device, dtype, size):
    """Logits hundreds apart: their exponentials are far beyond f32."""
    x, w, targets, grad = operands(TYPES[dtype], 40, 300, 64, 7)
    w = rounded(as_float64(w) * size, TYPES[dtype])
    check(forward(device, x, w, targets), cross_entropy(x, w, targets))
    # The gradients from the logits' own lse: an error of f32 in it would be one of
    # the whole distribution.
    lse = lse_of(x, w)
    check(backward(device, x, w, targets, lse, grad), cross_entropy_backward(x, w, targets, lse, grad))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 100])
def test_logits_that_are_no_numbers(device, dtype, rows):
    """Rows of x with a NaN have a loss that is one; words whose logits are minus
    infinity everywhere count for nothing."""
    x, w, targets, grad = operands(TYPES[dtype], rows, 90, 32, 8, left_out=0)
    x = rounded(np.abs(as_float64(x)) + 0.1, TYPES[dtype])
    w[3] = rounded(np.array([-np.inf]), TYPES[dtype])[0]
    targets[targets == 3] = 4
    x[2, 5] = rounded(np.array([np.nan]), TYPES[dtype])[0]
    got = forward(device, x, w, targets)
    assert np.isnan(got["loss"][2]) and np.isnan(got["lse"][2])
    rows_left = np.arange(rows) != 2
    w_left = np.delete(w, 3, 0)
    moved = np.where(targets > 3, targets - 1, targets).astype(np.uint32)
    value, bound = cross_entropy(x[rows_left], w_left, moved[rows_left])
    near(got["loss"][rows_left], value["loss"], bound["loss"], "loss")
    near(got["lse"][rows_left], value["lse"], bound["lse"], "lse")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [2.0**-120, 1.0, 2.0**100])
def test_gradients_of_any_size(device, dtype, size):
    x, w, targets, grad = operands(TYPES[dtype], 60, 130, 50, 9)
    grad = (grad * size).astype(np.float32)
    grad[5:9] = 0
    lse = lse_of(x, w)
    check(backward(device, x, w, targets, lse, grad), cross_entropy_backward(x, w, targets, lse, grad))


def test_like_gradients_cost_no_common_factor(device):
    """The gradients of a mean are all 1/n.  Rounded into G, such a factor would be
    off by the same part in every term: here by 2^-8.6 of all of them."""
    n = 354  # 1/354 lies 0.0026 of itself from the nearest of 8 bits
    x, w, targets, _ = operands(hx.bfloat16, n, 500, 64, 3, left_out=0)
    grad, lse = np.full(n, 1 / n, np.float32), lse_of(x, w)
    got = backward(device, x, w, targets, lse, grad)
    value, _ = cross_entropy_backward(x, w, targets, lse, grad)
    for name in got:
        scale = (as_float64(got[name]) * value[name]).sum() / (value[name] ** 2).sum()
        # Roundings at random, 2^-8 a term of thousands, even out.
        assert abs(scale - 1) <= 2.0**-11


@pytest.mark.parametrize("dtype", TYPES)
def test_vocabulary_in_pieces(device, dtype):
    """G of all rows passes what a piece may have: three pieces, the last one short."""
    rows, vocab, width = (70000, 4500, 8) if dtype == "bf16" else (35000, 4500, 8)
    x, w, targets, grad = operands(TYPES[dtype], rows, vocab, width, 11)
    lse = forward(device, x, w, targets)["lse"]
    got = backward(device, x, w, targets, lse, grad)
    part = np.arange(0, rows, 977)
    value, bound = cross_entropy_backward(x[part], w, targets[part], lse[part], grad[part])
    near(got["dx"][part], value["dx"], bound["dx"], "dx")
    total, off = np.zeros((vocab, width)), np.zeros((vocab, width))
    size = np.zeros((vocab, width))
    for lo in range(0, rows, 5000):
        rng = slice(lo, lo + 5000)
        value, bound = cross_entropy_backward(x[rng], w, targets[rng], lse[rng], grad[rng])
        total += value["dw"]
        off += bound["dw"]
        size += np.abs(value["dw"])
    # Of sums over 5000 rows a bound each; the whole sum is 14 times as long.
    near(got["dw"], total, 14 * off, "dw")


def test_empty(device):
    f = np.float32
    none, ops = device.alloc_zeroed(f, 0), hx.RocmLossOps()
    no_targets = device.alloc_zeroed(np.uint32, 0)
    no_rows = StridedView(none, Layout.c_contiguous([0, 4]))
    vw, _ = padded(device, np.ones((3, 4), f))
    vg, read = padded(device, np.ones((3, 4), f))
    ops.linear_cross_entropy_into(device, no_rows, vw, no_targets, none)
    ops.linear_cross_entropy_backward_into(device, no_rows, vw, no_targets, none, none, no_rows, vg)
    device.synchronize()
    assert not read().any()
    # No words: nothing to be a target.
    vx, _ = padded(device, np.ones((2, 4), f))
    vd, read = padded(device, np.ones((2, 4), f))
    no_words = StridedView(none, Layout.c_contiguous([0, 4]))
    two, at = vector(device, np.full(2, 7, f)), vector(device, np.zeros(2, np.uint32))
    lse = vector(device, np.zeros(2, f))
    ops.linear_cross_entropy_into(device, vx, no_words, at, two, lse)
    ops.linear_cross_entropy_backward_into(device, vx, no_words, at, lse, two, vd, no_words)
    device.synchronize()
    assert not device.download_owned(two).any() and np.all(device.download_owned(lse) == -np.inf) and not read().any()
    # No width: all words alike.
    thin, thin_w = (StridedView(none, Layout.c_contiguous([n, 0])) for n in (2, 3))
    ops.linear_cross_entropy_into(device, thin, thin_w, at, two)
    device.synchronize()
    assert np.abs(device.download_owned(two) - np.log(3)).max() <= 1e-6


@pytest.mark.parametrize("rows,vocab,width", [(4, 30, 20), (80, 100, 33)])
def test_gradient_against_differences(device, rows, vocab, width):
    x, w, targets, grad = operands(np.float32, rows, vocab, width, 12)
    got = forward(device, x, w, targets)
    back = backward(device, x, w, targets, got["lse"], grad)
    rng = np.random.default_rng(1)

    def loss(xx, ww):
        logits = xx @ ww.T
        top = logits.max(1, keepdims=True)
        lse = top[:, 0] + np.log(np.exp(logits - top).sum(1))
        has = targets < vocab
        return (grad * np.where(has, lse - logits[np.arange(rows), np.where(has, targets, 0)], 0)).sum()

    base = [v.astype(np.float64) for v in (x, w)]
    for i, name in enumerate(("dx", "dw")):
        way, h = rng.normal(size=base[i].shape), 1e-4
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + h * way, base[i] - h * way
        slope = (loss(*up) - loss(*down)) / (2 * h)
        size = np.abs(back[name].astype(np.float64) * way).sum()
        assert abs((back[name].astype(np.float64) * way).sum() - slope) <= 1e-5 * size + 1e-7


@pytest.mark.parametrize("dtype", TYPES)
def test_runs_repeat_to_the_bit(device, dtype):
    x, w, targets, grad = operands(TYPES[dtype], 600, 3000, 200, 4)
    first = forward(device, x, w, targets)
    back = backward(device, x, w, targets, first["lse"], grad)
    for _ in range(2):
        again = forward(device, x, w, targets)
        assert all(np.array_equal(first[k], again[k]) for k in first)
        again = backward(device, x, w, targets, first["lse"], grad)
        assert all(np.array_equal(back[k], again[k]) for k in back)
