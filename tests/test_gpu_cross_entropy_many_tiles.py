"""Losses whose product has more tiles than a launch has blocks."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from hephaestus_amd import Layout, StridedView
from layer_reference import EPS32, as_float64, padded, rounded, vector

pytestmark = pytest.mark.gpu


def test_more_tiles_than_a_launch_takes(device):
    """300 rows over 2^28 - 1 words are 10.5 million tiles of 64 x 128, two launches.  The
    words lie in one another, a dword apart, and repeat every 4096, so that the sum over
    all of them is one over 4096."""
    rows, vocab, width, period = 300, (1 << 28) - 1, 8, 4096
    rng = np.random.default_rng(5)
    x = rounded(rng.normal(size=(rows, width)), hx.bfloat16)
    pattern = rounded(rng.normal(size=2 * period), hx.bfloat16)
    w = device.upload(np.tile(pattern, vocab // period + 2)[:2 * (vocab - 1) + width])
    words = StridedView(w, Layout.try_new([vocab, width], [2, 1]))
    targets = rng.integers(0, vocab, rows).astype(np.uint32)
    # The words where one launch ends and the next begins, and the last ones.
    edge = ((1 << 23) - 8) // 5 * 128
    targets[:60] = np.clip(edge + np.arange(60) * 64 - 1800, 0, vocab - 1)
    targets[60:64] = vocab - 1 - np.arange(4)
    loss, lse = (vector(device, np.full(rows, 7, np.float32)) for _ in range(2))
    hx.RocmLossOps().linear_cross_entropy_into(device, padded(device, x)[0], words, vector(device, targets), loss, lse)
    device.synchronize()
    twice = as_float64(np.concatenate([pattern, pattern[:width]]))
    one = np.array([twice[2 * i:2 * i + width] for i in range(period)])
    logits = as_float64(x) @ one.T
    # 65536 times the period, but for its last word.
    total = np.exp(logits).sum(1) * (vocab // period + 1) - np.exp(logits[:, -1])
    want = np.log(total)
    # Each of 256 threads joins 8192 tiles in turn, two roundings each; the logits' and the
    # exponentials' own are those of the smaller losses.
    off = EPS32 * (2 * 8192 + 600 + 8 * np.abs(want)) + (width / 4 + 16) * EPS32 * (np.abs(as_float64(x)) @ np.abs(one).T).max(1)
    got = device.download_owned(lse)
    assert np.all(np.abs(got - want) <= off)
    picked = logits[np.arange(rows), targets % period]
    assert np.all(np.abs(device.download_owned(loss) - (want - picked)) <= 2 * off)



def test_the_most_rows(device):
    """2^28 - 1 rows that are one row in memory: the join's last block of 16 rows is past
    what one launch may have."""
    rows, vocab, width = (1 << 28) - 1, 50, 8
    rng = np.random.default_rng(7)
    x, w = rounded(rng.normal(size=(1, width)), hx.bfloat16), rounded(rng.normal(size=(vocab, width)), hx.bfloat16)
    same = StridedView(device.upload(x), Layout.try_new([rows, width], [0, 1]))
    targets = device.alloc_zeroed(np.uint32, rows)
    some = np.unique(np.concatenate([np.arange(40), rows - 1 - np.arange(40), rng.integers(0, rows, 40)]))
    kinds = rng.integers(0, vocab + 1, len(some)).astype(np.uint32)  # `vocab` leaves a row out
    for at, kind in zip(some, kinds):
        device.write_sub_buffer(targets, int(at), np.array([kind], np.uint32))
    loss = device.alloc_uninitialized(np.float32, rows)
    hx.RocmLossOps().linear_cross_entropy_into(device, same, padded(device, w)[0], targets, loss)
    device.synchronize()
    logits = (as_float64(x) @ as_float64(w).T)[0]
    want = np.append(np.log(np.exp(logits).sum()) - logits, 0.0)
    off = EPS32 * (600 + 8 * np.abs(want).max()) + 2 * (width / 4 + 16) * EPS32 * (np.abs(as_float64(x)) @ np.abs(as_float64(w)).T).max()
    got = device.download_owned(loss)
    assert np.abs(got[some] - want[kinds]).max() <= off
    got[some] = got[100]
    assert abs(float(got[100]) - want[0]) <= off and np.all(got == got[100])
