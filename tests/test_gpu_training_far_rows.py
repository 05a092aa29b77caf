"""Rows of norms and losses that lie 2^32 bytes and more into their buffers, read and
written."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from hephaestus_amd import NO_TARGET, Layout, StridedView
from layer_reference import rounded, vector
from test_gpu_cross_entropy import lse_of, operands as loss_operands
from test_gpu_layer_norm import EPSILON, operands as norm_operands, stats_of
from training_reference import TYPES, cross_entropy, cross_entropy_backward, layer_norm, layer_norm_backward, near

pytestmark = pytest.mark.gpu

FAR = (1 << 32) + 192  # bytes from the first row to the last


class FarRows:
    """A view of rows whose last one begins FAR bytes past the first, in a buffer that
    holds nothing else."""

    def __init__(self, device, rows, cols, dtype, values=None):
        self.device, self.dtype, self.rows, self.cols = device, np.dtype(dtype), rows, cols
        size = 2 if dtype == hx.bfloat16 else 4
        self.step = -(-FAR // size // (rows - 1) // 8) * 8
        self.pool = device.alloc_uninitialized(dtype, self.step * (rows - 1) + cols)
        assert self.step * (rows - 1) * size >= 1 << 32
        self.view = StridedView(self.pool, Layout.try_new([rows, cols], [self.step, 1]))
        if values is not None:
            for i, row in enumerate(values):
                device.write_sub_buffer(self.pool, i * self.step, row)

    def read(self):
        size = self.pool.itemsize
        rows = [self.device.download_owned(self.device.borrow(self.pool.ptr + i * self.step * size, self.dtype, self.cols,
                                                              self.pool)) for i in range(self.rows)]
        return np.stack(rows)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [300, 40000])
def test_norm(device, dtype, cols):
    t, rows = TYPES[dtype], 5
    x, r, w, b, dy, past = norm_operands(t, rows, cols, 3)
    far = {name: FarRows(device, rows, cols, t, v) for name, v in (("x", x), ("r", r))}
    out = {name: FarRows(device, rows, cols, t) for name in ("y", "h")}
    ops = hx.RocmLayerNormOps()
    ops.layer_norm_into(device, far["x"].view, vector(device, w), vector(device, b), EPSILON, out["y"].view,
                        residual=far["r"].view, residual_out=out["h"].view)
    device.synchronize()
    value, bound = layer_norm(x, r, w, b, EPSILON)
    for name in out:
        near(out[name].read(), value[name], bound[name], name)
    mean, rstd = stats_of(x)
    far_dy, far_past = FarRows(device, rows, cols, t, dy), FarRows(device, rows, cols, t, past)
    dw = vector(device, np.zeros(cols, np.float32))
    ops.layer_norm_backward_into(device, far_dy.view, far["x"].view, vector(device, w), vector(device, mean),
                                 vector(device, rstd), out["y"].view, residual_grad=far_past.view, grad_weight=dw)
    device.synchronize()
    value, bound = layer_norm_backward(dy, x, w, mean, rstd, past)
    near(out["y"].read(), value["dh"], bound["dh"], "dh")
    near(device.download_owned(dw), value["dw"], bound["dw"], "dw")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,width", [(5, 70, 64), (300, 3, 33)])
def test_loss(device, dtype, rows, vocab, width):
    t = TYPES[dtype]
    x, w, targets, grad = loss_operands(t, rows, vocab, width, 5)
    targets[0], targets[1] = NO_TARGET, vocab - 1
    fx, fw = FarRows(device, rows, width, t, x), FarRows(device, vocab, width, t, w)
    loss, lse = (vector(device, np.zeros(rows, np.float32)) for _ in range(2))
    ops, at = hx.RocmLossOps(), vector(device, targets)
    ops.linear_cross_entropy_into(device, fx.view, fw.view, at, loss, lse)
    dx, dw = FarRows(device, rows, width, t), FarRows(device, vocab, width, t)
    from_lse = lse_of(x, w)
    ops.linear_cross_entropy_backward_into(device, fx.view, fw.view, at, vector(device, from_lse), vector(device, grad),
                                           dx.view, dw.view)
    device.synchronize()
    value, bound = cross_entropy(x, w, targets)
    near(device.download_owned(loss), value["loss"], bound["loss"], "loss")
    near(device.download_owned(lse), value["lse"], bound["lse"], "lse")
    value, bound = cross_entropy_backward(x, w, targets, from_lse, grad)
    near(dx.read(), value["dx"], bound["dx"], "dx")
    near(dw.read(), value["dw"], bound["dw"], "dw")


def test_norm_rows_backwards_from_far(device):
    """A negative stride from the last row on."""
    t, rows, cols = np.float32, 3, 260
    x, _, w, b, _, _ = norm_operands(t, rows, cols, 4)
    far, out = FarRows(device, rows, cols, t, x), FarRows(device, rows, cols, t)
    back = StridedView(far.pool, Layout.try_new([rows, cols], [-far.step, 1], far.step * (rows - 1)))
    hx.RocmLayerNormOps().layer_norm_into(device, back, vector(device, w), vector(device, b), EPSILON, out.view)
    device.synchronize()
    value, bound = layer_norm(x[::-1], None, w, b, EPSILON)
    near(out.read(), value["y"], bound["y"], "y")
