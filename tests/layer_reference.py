"""The layer operators written out plainly in 64 bits, and the tolerances of
their tests."""
from __future__ import annotations

import math

import numpy as np

import hephaestus_amd as hx
from hephaestus_amd import Layout, StridedView

EPS32 = 2.0**-24   # half a unit in the last place of f32, relative
EPS16 = 2.0**-8    # the same of bf16, which keeps 8 bits


def as_float64(array):
    array = np.asarray(array)
    return (hx.float32_from_bfloat16(array) if array.dtype == hx.bfloat16 else array).astype(np.float64)


def rounded(values, dtype):
    """Values of an element type, as the device takes them."""
    if dtype == hx.bfloat16:
        return hx.bfloat16_from_float32(np.asarray(values, np.float32))
    return np.asarray(values, np.float32)


def norm_quantize(x, residual, weight, epsilon):
    """(h, y / s before rounding, s) in 64 bits."""
    h = as_float64(x) + (0.0 if residual is None else as_float64(residual))
    y = h / np.sqrt(np.mean(h * h, axis=1, keepdims=True) + epsilon) * as_float64(weight)
    s = np.max(np.abs(y), axis=1) / 127
    return h, np.divide(y, s[:, None], out=np.zeros_like(y), where=s[:, None] > 0), s


def matmul_i8(a, b, sa, sb):
    return sa.astype(np.float64)[:, None] * (a.astype(np.int64) @ b.astype(np.int64).T) * sb.astype(np.float64)


def linear_attention(q, k, v, log_decay, scale, state=None, lengths=None):
    """The recurrence, token by token: (out, state after the last token, the
    same with every term's magnitude, by which errors are measured)."""
    q, k, v = as_float64(q), as_float64(k), as_float64(v)
    batch, tokens, heads, dk = q.shape
    dv, group = v.shape[3], heads // max(1, k.shape[2])
    out = np.zeros((batch, tokens, heads, dv))
    size = np.zeros_like(out)
    first = np.zeros((batch, heads, dk, dv)) if state is None else state.astype(np.float64)
    last, last_size = first.copy(), np.abs(first)
    decay = np.exp(np.asarray(log_decay, np.float64))
    for b in range(batch):
        for h in range(heads):
            for t in range(tokens if lengths is None else min(tokens, int(lengths[b]))):
                kt, vt = k[b, t, h // group], v[b, t, h // group]
                last[b, h] = decay[h] * last[b, h] + np.outer(kt, vt)
                last_size[b, h] = decay[h] * last_size[b, h] + np.abs(np.outer(kt, vt))
                out[b, t, h] = scale * (q[b, t, h] @ last[b, h])
                size[b, t, h] = abs(scale) * (np.abs(q[b, t, h]) @ last_size[b, h])
    return out, last, size, last_size


def padded(dev, array, strides_pad=0, offset=0, order=None):
    """A device view of `array` whose outermost memory dimension rows are
    `strides_pad` elements apart beyond the dense ones and which begins `offset`
    elements into its buffer.  `order` lists the dimensions from the outermost in
    memory; the last stays last.  Returns (view, read), where read() downloads
    the view's values."""
    array = np.asarray(array)
    order = tuple(order or range(array.ndim))
    dense = np.ascontiguousarray(array.transpose(order))
    strides, step = [0] * array.ndim, 1
    for d in reversed(order):
        strides[d] = step
        step *= max(1, array.shape[d]) if d != order[-1] else max(1, array.shape[d]) + strides_pad
    length = offset + max(1, step)
    filler = np.zeros(length, array.dtype)
    if array.dtype != hx.bfloat16 and array.dtype.kind == "f":
        filler[:] = np.nan  # what lies between the rows must not be read into a result
    elif array.dtype == hx.bfloat16:
        filler = np.full(length, 0x7FC0, np.uint16).view(hx.bfloat16)
    elif array.dtype == np.int8:
        filler[:] = 99
    host = filler.copy()
    spread = np.lib.stride_tricks.as_strided(host[offset:], dense.shape, [strides[d] * host.itemsize for d in order])
    if array.size:
        spread[...] = dense
    buffer = dev.upload(host)
    view = StridedView(buffer, Layout.try_new(array.shape, strides, offset))

    def read():
        got = dev.download_owned(buffer)
        part = np.lib.stride_tricks.as_strided(got[offset:], dense.shape,
                                               [strides[d] * got.itemsize for d in order]).copy()
        # Nothing outside the view was written.
        np.lib.stride_tricks.as_strided(got[offset:], dense.shape, [strides[d] * got.itemsize for d in order])[
            ...] = dense
        np.lib.stride_tricks.as_strided(host[offset:], dense.shape, [strides[d] * host.itemsize for d in order])[
            ...] = dense
        assert got.tobytes() == host.tobytes(), "elements outside the view were written"
        return part.transpose(np.argsort(order))

    return view, read


def vector(dev, values):
    return dev.upload(np.ascontiguousarray(values))


def sqrt_size(terms):
    return math.sqrt(max(1, terms))
