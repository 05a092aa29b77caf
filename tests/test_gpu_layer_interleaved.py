"""Layer operators on views that lie between one another in one buffer."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
import test_gpu_linear_attention as attention
import test_gpu_matmul_i8 as matmul
import test_gpu_norm_quantize as norm

pytestmark = pytest.mark.gpu

N = hx.Layout.try_new
TYPES = attention.TYPES


def spread(host, layout):
    """The elements of a host buffer that a layout names."""
    strides = [s * host.itemsize for s in layout.strides]
    return np.lib.stride_tricks.as_strided(host[layout.offset:], layout.shape, strides)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 5, 70, 1500])
@pytest.mark.parametrize("dk,dv,extra", [(64, 64, 0), (37, 53, 3)])
def test_outputs_beside_q_k_and_v(device, dtype, tokens, dk, dv, extra):
    """Rows of q | k | v | o, and a pool with two slots of state a sequence."""
    t, heads, batch = TYPES[dtype], 3, 2
    q, k, v, decay, state = attention.operands(t, batch, tokens, heads, heads, dk, dv, 41)
    row = 2 * heads * (dk + dv) + extra
    at, layouts = 0, []
    for width in (dk, dk, dv, dv):
        layouts.append(N([batch, tokens, heads, width], [tokens * row, row, width, 1], at))
        at += heads * width
    host = np.zeros(batch * tokens * row, t)
    for layout, x in zip(layouts, (q, k, v)):
        spread(host, layout)[...] = x
    rows = device.upload(host)
    slots = [N([batch, heads, dk, dv], [2 * heads * dk * dv, dk * dv, dv, 1], i * heads * dk * dv) for i in range(2)]
    pool = np.full(2 * batch * heads * dk * dv, 5, np.float32)
    spread(pool, slots[0])[...] = state
    states = device.upload(pool)
    vq, vk, vv, vo = (hx.StridedView(rows, layout) for layout in layouts)
    hx.RocmLinearAttentionOps().linear_attention_into(
        device, vq, vk, vv, device.upload(decay), vo, state_in=hx.StridedView(states, slots[0]),
        state_out=hx.StridedView(states, slots[1]))
    device.synchronize()
    got, got_pool = device.download_owned(rows), device.download_owned(states)
    attention.check(q, k, v, decay, state, None, (spread(got, layouts[3]).copy(), spread(got_pool, slots[1]).copy()))
    assert np.array_equal(spread(got_pool, slots[0]), state)
    spread(got, layouts[3])[...] = np.zeros(1, t)
    assert got.tobytes() == host.tobytes()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [61, 4096, 40000])
def test_rows_in_turn(device, dtype, cols):
    """x, the residual and h take turns in the rows of one buffer."""
    t = TYPES[dtype]
    rng = np.random.default_rng(cols)
    x, r = (norm.rounded(rng.normal(size=(5, cols)), t) for _ in range(2))
    w = norm.rounded(rng.uniform(0.5, 2, cols), t)
    layouts = [N([5, cols], [3 * cols, 1], i * cols) for i in range(3)]
    host = np.zeros(15 * cols, t)
    spread(host, layouts[0])[...], spread(host, layouts[1])[...] = x, r
    rows = device.upload(host)
    views = [hx.StridedView(rows, layout) for layout in layouts]
    q, scales = device.alloc_zeroed(np.int8, 5 * cols), device.alloc_zeroed(np.float32, 5)
    hx.RocmNormOps().rms_norm_quantize_into(device, views[0], device.upload(w), norm.EPSILON,
                                            hx.StridedView(q, hx.Layout.c_contiguous([5, cols])), scales,
                                            residual=views[1], residual_out=views[2])
    device.synchronize()
    got = device.download_owned(rows)
    norm.check(x, r, w, (spread(got, layouts[2]).copy(), device.download_owned(q).reshape(5, cols),
                         device.download_owned(scales)))
    spread(got, layouts[2])[...] = np.zeros(1, t)
    assert got.tobytes() == host.tobytes()


@pytest.mark.parametrize("m,n,k,gap", [(3, 50, 200, 0), (20, 64, 130, 2), (90, 70, 256, 0), (300, 520, 129, 3)])
def test_products_between_the_rows_of_an_operand(device, m, n, k, gap):
    """Each row of a is followed by the row of the output that it gives."""
    a, b, sa, sb = matmul.operands(m, n, k, 42)
    first = -(-(k + gap) // 4) * 4  # the output's rows begin on f32 boundaries
    pitch = first + 4 * n
    host = np.full(m * pitch, 99, np.int8)
    la = N([m, k], [pitch, 1])
    spread(host, la)[...] = a
    rows = device.upload(host)
    lo = N([m, n], [pitch // 4, 1], first // 4)
    floats = device.borrow(rows.ptr, np.float32, m * pitch // 4, owner=rows)
    hx.RocmMatrixOps().matmul_i8_into(device, hx.StridedView(rows, la), device.upload(sa),
                                      hx.StridedView(device.upload(b), hx.Layout.c_contiguous([n, k])), device.upload(sb),
                                      hx.StridedView(floats, lo))
    device.synchronize()
    got = device.download_owned(rows)
    matmul.check(a, b, sa, sb, spread(got.view(np.float32), lo).copy())
    spread(got.view(np.float32), lo)[...] = spread(host.view(np.float32), lo)
    assert got.tobytes() == host.tobytes()
