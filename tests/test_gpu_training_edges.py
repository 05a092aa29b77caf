"""Training operators where their launches meet: ends of tiles, of steps and of parts."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
import test_gpu_cross_entropy as entropy
import test_gpu_gated_recurrence as recurrence
from hephaestus_amd import NO_TARGET
from layer_reference import as_float64, padded, rounded, vector
from training_reference import TYPES, cross_entropy, cross_entropy_backward, gated_recurrence

pytestmark = pytest.mark.gpu

# Few tiles, logits in parts of the width; one part; a last step of whole 16 bytes, of
# some, and none.
WIDTHS = [(5, 90, 2100), (5, 90, 2112), (130, 700, 64), (130, 700, 72), (130, 700, 70), (300, 260, 136)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,width", WIDTHS)
def test_words_of_minus_infinity(device, dtype, rows, vocab, width):
    """They count for nothing, wherever a step of the width ends."""
    x, w, targets, _ = entropy.operands(TYPES[dtype], rows, vocab, width, width)
    x = rounded(np.abs(as_float64(x)) + 0.1, TYPES[dtype])
    gone = [0, vocab // 2, vocab - 1]
    w[gone] = rounded(np.array([-np.inf]), TYPES[dtype])[0]
    targets[np.isin(targets, gone)] = 1
    got = entropy.forward(device, x, w, targets)
    place = np.cumsum(~np.isin(np.arange(vocab), gone)) - 1
    moved = np.where(targets < vocab, place[np.minimum(targets, vocab - 1)], NO_TARGET).astype(np.uint32)
    entropy.check(got, cross_entropy(x, np.delete(w, gone, 0), moved))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,width", WIDTHS)
def test_logits_that_are_no_numbers_stay_in_their_rows(device, dtype, rows, vocab, width):
    x, w, targets, grad = entropy.operands(TYPES[dtype], rows, vocab, width, width + 1)
    clean = entropy.forward(device, x, w, targets)
    x[1, width - 1] = rounded(np.array([np.nan]), TYPES[dtype])[0]
    targets[1] = 0
    got = entropy.forward(device, x, w, targets)
    left = np.arange(rows) != 1
    for name in got:
        assert np.isnan(got[name][1]) and np.array_equal(got[name][left], clean[name][left])
    # Left out, the row adds nothing to the gradients.
    targets[1] = NO_TARGET
    back = entropy.backward(device, x, w, targets, got["lse"], grad)
    plain = as_float64(x)
    plain[1] = 0.0
    lse = np.where(left, got["lse"], 0.0).astype(np.float32)
    entropy.check(back, cross_entropy_backward(rounded(plain, TYPES[dtype]), w, targets, lse, grad))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,width", WIDTHS)
@pytest.mark.parametrize("which", ["first", "last", "none"])
def test_one_target_for_all_rows(device, dtype, rows, vocab, width, which):
    x, w, targets, grad = entropy.operands(TYPES[dtype], rows, vocab, width, width + 2)
    targets[:] = {"first": 0, "last": vocab - 1, "none": NO_TARGET}[which]
    got = entropy.forward(device, x, w, targets)
    entropy.check(got, cross_entropy(x, w, targets))
    back = entropy.backward(device, x, w, targets, got["lse"], grad)
    entropy.check(back, cross_entropy_backward(x, w, targets, got["lse"], grad))
    if which == "none":
        assert not got["loss"].any() and not as_float64(back["dx"]).any() and not as_float64(back["dw"]).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", [6, 65, 130])
def test_lengths_about_the_parts_with_the_state_in_place(device, dtype, channels):
    lengths = [0, 1, 63, 64, 65, 128, 129, 400]
    gate, x, _, first, _ = recurrence.operands(TYPES[dtype], len(lengths), 400, channels, channels)
    state, read = padded(device, first, 3)
    out, read_h = padded(device, rounded(np.full(x.shape, 9.0), TYPES[dtype]))
    hx.RocmRecurrenceOps().gated_recurrence_into(
        device, padded(device, gate)[0], padded(device, x)[0], out, state_in=state, state_out=state,
        lengths=vector(device, np.array(lengths, np.uint32)))
    device.synchronize()
    recurrence.check({"h": read_h(), "last": read()}, gated_recurrence(gate, x, first, lengths))


def test_products_in_parts_repeat_to_the_bit(device):
    """Two sizes in turn, which share their stream's scratch."""
    results = []
    for turn in range(3):
        for rows, vocab, width in ((5, 90, 2100), (40, 2050, 4200)):
            x, w, targets, grad = entropy.operands(np.float32, rows, vocab, width, rows)
            got = entropy.forward(device, x, w, targets)
            back = entropy.backward(device, x, w, targets, got["lse"], grad)
            results.append([got["loss"].tobytes(), got["lse"].tobytes(), back["dx"].tobytes(), back["dw"].tobytes()])
    assert results[0::2] == [results[0]] * 3 and results[1::2] == [results[1]] * 3
