"""Products of 8-bit integers with scales against exact integer sums."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from layer_reference import EPS16, EPS32, as_float64, matmul_i8, padded, rounded, vector

pytestmark = pytest.mark.gpu

TYPES = {"f32": np.float32, "bf16": hx.bfloat16}


def operands(m, n, k, seed=0):
    rng = np.random.default_rng(seed * 7919 + m * 31 + n * 17 + k)
    a, b = (rng.integers(-128, 128, (rows, k), dtype=np.int8) for rows in (m, n))
    sa, sb = (rng.uniform(0.001, 0.1, rows).astype(np.float32) for rows in (m, n))
    return a, b, sa, sb


def run(device, a, b, sa, sb, dtype, *, pad=0, offset=0, prepared=False):
    va, _ = padded(device, a, pad, offset)
    vb, _ = padded(device, b, pad and pad + 1, offset)
    vo, read = padded(device, rounded(np.full((a.shape[0], b.shape[0]), 7.0), dtype), pad, offset)
    args = (device, va, vector(device, sa), vb, vector(device, sb), vo)
    if prepared:
        plan = hx.RocmMatrixOps().prepare_matmul_i8(*args)
        for _ in range(3):  # a plan's workspace serves every dispatch
            plan.dispatch()
    else:
        hx.RocmMatrixOps().matmul_i8_into(*args)
    device.synchronize()
    return read()


def check(a, b, sa, sb, got):
    want = matmul_i8(a, b, sa, sb)
    # The sum as f32, two products, and the output's own rounding.
    bound = 4 * EPS32 + (EPS16 if got.dtype == hx.bfloat16 else 0)
    assert np.all(np.abs(as_float64(got) - want) <= np.abs(want) * bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 1, 64), (1, 17, 5), (2, 16, 64), (3, 5, 63), (4, 33, 65), (1, 64, 128), (1, 256, 4096),
    (1, 1000, 1000), (5, 300, 2000), (15, 64, 256), (16, 64, 256), (17, 65, 257), (31, 100, 512), (32, 1024, 1024),
    (33, 250, 130), (48, 512, 384), (64, 2048, 1024), (63, 127, 1023), (65, 129, 320), (100, 100, 100),
    (127, 255, 127), (128, 128, 128), (129, 257, 129), (200, 1000, 4099), (256, 256, 256), (255, 257, 640),
    (512, 768, 1024), (1000, 1027, 515), (2000, 64, 96), (64, 2000, 48), (300, 16, 16)])
def test_sizes(device, dtype, m, n, k):
    ops = operands(m, n, k)
    check(*ops, run(device, *ops, TYPES[dtype]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,offset", [(1, 0), (4, 1), (16, 16), (5, 3), (64, 8)])
@pytest.mark.parametrize("m,n,k", [(1, 100, 320), (20, 64, 500), (70, 300, 256), (260, 270, 384)])
def test_strides_and_offsets(device, dtype, pad, offset, m, n, k):
    ops = operands(m, n, k, 1)
    check(*ops, run(device, *ops, TYPES[dtype], pad=pad, offset=offset, prepared=True))


@pytest.mark.parametrize("m,n,k", [(8192, 64, 64), (3, 8192, 64), (1024, 1024, 1024), (1500, 2500, 704)])
def test_many_tiles(device, m, n, k):
    ops = operands(m, n, k, 2)
    check(*ops, run(device, *ops, hx.bfloat16))


@pytest.mark.parametrize("m,n", [(1, 40), (40, 40), (300, 300)])
@pytest.mark.parametrize("k", [131071, 100000])
def test_the_longest_sums(device, m, n, k):
    """The largest magnitudes at the greatest depth: sums just inside int32."""
    a, b = np.full((m, k), -128, np.int8), np.full((n, k), -128, np.int8)
    b[::2] = 127
    sa, sb = np.full(m, 0.5, np.float32), np.linspace(1, 2, n).astype(np.float32)
    got = run(device, a, b, sa, sb, np.float32)
    sums = np.where(np.arange(n) % 2 == 0, -128 * 127 * k, 128 * 128 * k).astype(np.float64)
    want = 0.5 * sums * sb.astype(np.float64)
    assert np.all(np.abs(got - want) <= np.abs(want) * 4 * EPS32)


def test_rows_reversed_and_broadcast(device):
    """A negative stride in a, one row of b for every channel."""
    a, b, sa, sb = operands(50, 1, 200, 3)
    sb = np.linspace(0.1, 1, 70).astype(np.float32)
    out = device.alloc_zeroed(np.float32, 50 * 70)
    hx.RocmMatrixOps().matmul_i8_into(
        device, hx.StridedView(device.upload(a), hx.Layout.try_new([50, 200], [-200, 1], 49 * 200)), device.upload(sa),
        hx.StridedView(device.upload(b), hx.Layout.try_new([70, 200], [0, 1])), device.upload(sb),
        hx.StridedView(out, hx.Layout.try_new([50, 70], [-70, 1], 49 * 70)))
    device.synchronize()
    check(a[::-1], np.repeat(b, 70, 0), sa, sb, device.download_owned(out).reshape(50, 70)[::-1])


def test_empty_operands(device):
    for m, n, k in ((0, 5, 8), (5, 0, 8), (3, 4, 0)):
        a, b, sa, sb = operands(m, n, k)
        got = run(device, a, b, sa, sb, np.float32)
        assert got.shape == (m, n) and not got.any()


def test_scales_that_are_not_numbers_stay_in_their_row_and_column(device):
    a, b, sa, sb = operands(70, 80, 128, 4)
    sa[3], sb[11] = np.nan, np.inf
    got = run(device, a, b, sa, sb, np.float32)
    assert np.isnan(got[3]).all()
    rest = np.delete(got, 3, 0)
    assert np.isinf(rest[:, 11]).all()
    assert np.isfinite(np.delete(rest, 11, 1)).all()


def test_same_bits_every_run(device):
    ops = operands(40, 600, 8192, 5)
    first = run(device, *ops, np.float32)
    for _ in range(3):
        assert first.tobytes() == run(device, *ops, np.float32, prepared=True).tobytes()


@pytest.mark.parametrize("k", [1, 15, 17, 129, 1500, 4099])
@pytest.mark.parametrize("m,n", [(17, 3), (33, 260)])
def test_rows_off_dwords(device, m, n, k):
    """Rows copied end to end: a block's part of the copy crosses rows and the
    border of a and b."""
    ops = operands(m, n, k, 7)
    check(*ops, run(device, *ops, np.float32, pad=1, offset=1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad,offset", [(0, 0), (2, 1), (1, 2), (3, 3)])
@pytest.mark.parametrize("m,n,k", [(1, 16, 127), (15, 40, 1025), (16, 33, 4099), (17, 100, 129), (31, 70, 2047),
                                   (32, 8200, 257), (32, 33, 4097), (33, 33, 1023)])
def test_few_tokens_off_dwords(device, dtype, m, n, k, pad, offset):
    """Each row at its own address modulo 4; both sides of the bounds on tokens,
    channels and depth."""
    ops = operands(m, n, k, 8)
    check(*ops, run(device, *ops, TYPES[dtype], pad=pad, offset=offset, prepared=True))
