"""Products of 8-bit integers with more channels or tokens than a launch takes."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from layer_reference import EPS16, EPS32, as_float64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,offset", [(1, 2**28 + 21, 0), (2, 2**27 + 5, 1), (3 * 2**26 + 9, 1, 0)])
def test_more_rows_than_a_launch_takes(device, m, n, offset):
    """Few tokens with rows on dwords and off them, and tiles; one row of either
    operand for all of its tokens or channels, its scales all its own."""
    rng = np.random.default_rng(m)
    a, b = (rng.integers(-128, 128, 8 + offset, dtype=np.int8) for _ in range(2))
    sa = ((np.arange(m) * 5) % 241 + 1).astype(np.float32)
    sb = ((np.arange(n) * 7) % 251 + 1).astype(np.float32)
    va = hx.StridedView(device.upload(a), hx.Layout.try_new([m, 8], [0, 1], offset))
    vb = hx.StridedView(device.upload(b), hx.Layout.try_new([n, 8], [0, 1], offset))
    out = device.alloc_zeroed(hx.bfloat16, m * n)
    hx.RocmMatrixOps().matmul_i8_into(device, va, device.upload(sa), vb, device.upload(sb),
                                      hx.StridedView(out, hx.Layout.c_contiguous([m, n])))
    device.synchronize()
    got = device.download_owned(out).reshape(m, n)
    out.free()
    total = int(a[offset:].astype(np.int64) @ b[offset:].astype(np.int64))
    assert total != 0
    for i in range(0, m, 2**25):
        for j in range(0, n, 2**25):
            want = total * sa[i:i + 2**25, None].astype(np.float64) * sb[j:j + 2**25]
            off = np.abs(as_float64(got[i:i + 2**25, j:j + 2**25]) - want)
            assert np.all(off <= np.abs(want) * (4 * EPS32 + EPS16)), (i, j)
