"""What the layer operators refuse, and in which words.  Checks run before a
device is touched, so these need none (the calls go to a device that was never
opened)."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from hephaestus_amd import Layout, RocmBuffer, StridedView

L, N = Layout.c_contiguous, Layout.try_new


class NoDevice:
    handle = None


def buffer(ptr, length, dtype):
    return RocmBuffer(None, ptr, length, dtype)


def view(ptr, layout, dtype, length=None):
    size = int(np.prod(layout.shape)) if length is None else length
    return StridedView(buffer(ptr, size, dtype), layout)


def norm(**change):
    a = {"x": view(0x1000000, L([4, 64]), np.float32), "weight": buffer(0x2000000, 64, np.float32), "epsilon": 1e-5,
         "quantized": view(0x3000000, L([4, 64]), np.int8), "scales": buffer(0x4000000, 4, np.float32),
         "residual": view(0x5000000, L([4, 64]), np.float32), "residual_out": view(0x6000000, L([4, 64]), np.float32)}
    a.update(change)
    hx.RocmNormOps().rms_norm_quantize_into(NoDevice, **a)


def matmul(**change):
    a = {"a": view(0x1000000, L([4, 64]), np.int8), "a_scales": buffer(0x2000000, 4, np.float32),
         "b": view(0x3000000, L([6, 64]), np.int8), "b_scales": buffer(0x4000000, 6, np.float32),
         "output": view(0x5000000, L([4, 6]), np.float32)}
    a.update(change)
    hx.RocmMatrixOps().matmul_i8_into(NoDevice, **a)


def attention(**change):
    f = np.float32
    a = {"q": view(0x1000000, L([2, 5, 4, 8]), f), "k": view(0x2000000, L([2, 5, 2, 8]), f),
         "v": view(0x3000000, L([2, 5, 2, 16]), f), "log_decay": buffer(0x4000000, 4, f),
         "output": view(0x5000000, L([2, 5, 4, 16]), f), "state_in": view(0x6000000, L([2, 4, 8, 16]), f),
         "state_out": view(0x7000000, L([2, 4, 8, 16]), f), "lengths": buffer(0x8000000, 2, np.uint32)}
    a.update(change)
    hx.RocmLinearAttentionOps().linear_attention_into(NoDevice, **a)


F, B, I8 = np.float32, hx.bfloat16, np.int8

REFUSED = [
    # norm: types, sizes, strides, storage
    (norm, {"x": view(0x1000000, L([4, 64]), np.int32)}, hx.InvalidConfiguration, "must be float32 or bfloat16"),
    (norm, {"weight": buffer(0x2000000, 64, B)}, hx.InvalidConfiguration, "norm weight must be float32"),
    (norm, {"residual": view(0x5000000, L([4, 64]), B)}, hx.InvalidConfiguration, "residual must be float32"),
    (norm, {"quantized": view(0x3000000, L([4, 64]), np.uint8)}, hx.InvalidConfiguration, "quantized output must be int8"),
    (norm, {"epsilon": -1.0}, hx.InvalidConfiguration, "epsilon"),
    (norm, {"epsilon": float("nan")}, hx.InvalidConfiguration, "epsilon"),
    (norm, {"weight": buffer(0x2000000, 63, F)}, hx.LengthMismatch, "64"),
    (norm, {"scales": buffer(0x4000000, 5, F)}, hx.LengthMismatch, "4"),
    (norm, {"x": view(0x1000000, L([256]), F)}, hx.DispatchFailed, "rank-2"),
    (norm, {"residual": view(0x5000000, L([4, 63]), F)}, hx.DispatchFailed, "residual has shape"),
    (norm, {"x": view(0x1000000, N([4, 64], [128, 2]), F, 512)}, hx.DispatchFailed, "contiguous last dimension"),
    (norm, {"x": view(0x1000000, L([4, 64]), F, 255)}, hx.DispatchFailed, "layout rejected"),
    (norm, {"x": view(0, L([4, 64]), F)}, hx.DispatchFailed, "null"),
    (norm, {"x": view(0x1000002, L([4, 64]), F)}, hx.DispatchFailed, "not aligned"),
    (norm, {"quantized": view(0x3000000, N([4, 64], [0, 1]), I8)}, hx.DispatchFailed, "reach an element twice"),
    (norm, {"quantized": view(0x3000000, N([4, 64], [63, 1]), I8)}, hx.DispatchFailed, "reach an element twice"),
    # norm: overlaps
    (norm, {"quantized": view(0x1000000, L([4, 64]), I8)}, hx.DispatchFailed, "must not overlap the norm input"),
    (norm, {"quantized": view(0x6000010, L([4, 64]), I8)}, hx.DispatchFailed, "must not overlap"),
    (norm, {"scales": buffer(0x2000010, 4, F)}, hx.DispatchFailed, "must not overlap the norm weight"),
    (norm, {"residual_out": view(0x1000100, L([4, 64]), F)}, hx.DispatchFailed, "be the view of the norm input"),
    (norm, {"residual_out": view(0x5000000, N([4, 64], [-64, 1], 192), F)}, hx.DispatchFailed,
     "be the view of the residual"),
    # matmul
    (matmul, {"a": view(0x1000000, L([4, 64]), F)}, hx.InvalidConfiguration, "operand a must be int8"),
    (matmul, {"b_scales": buffer(0x4000000, 6, B)}, hx.InvalidConfiguration, "scales of b must be float32"),
    (matmul, {"output": view(0x5000000, L([4, 6]), np.int32)}, hx.InvalidConfiguration, "float32 or bfloat16"),
    (matmul, {"b": view(0x3000000, L([6, 63]), I8)}, hx.DispatchFailed, "matmul b has shape"),
    (matmul, {"output": view(0x5000000, L([6, 4]), F)}, hx.DispatchFailed, "matmul output has shape"),
    (matmul, {"a_scales": buffer(0x2000000, 3, F)}, hx.LengthMismatch, "4"),
    (matmul, {"a": view(0x1000000, N([4, 64], [1, 4]), I8)}, hx.DispatchFailed, "contiguous last dimension"),
    (matmul, {"a": view(0x1000000, L([4, 131072]), I8), "b": view(0x3000000, L([6, 131072]), I8)}, hx.DispatchFailed,
     "exceeds the 32-bit sums"),
    (matmul, {"output": view(0x5000000, N([4, 6], [0, 1]), F)}, hx.DispatchFailed, "reach an element twice"),
    (matmul, {"output": view(0x3000000, L([4, 6]), F)}, hx.DispatchFailed, "must not overlap matmul b"),
    (matmul, {"output": view(0x2000008, L([4, 6]), F)}, hx.DispatchFailed, "must not overlap the scales of a"),
    # attention
    (attention, {"q": view(0x1000000, L([2, 5, 4, 8]), np.float64)}, hx.InvalidConfiguration, "float32 or bfloat16"),
    (attention, {"k": view(0x2000000, L([2, 5, 2, 8]), B)}, hx.InvalidConfiguration, "attention key must be float32"),
    (attention, {"log_decay": buffer(0x4000000, 4, B)}, hx.InvalidConfiguration, "log decay must be float32"),
    (attention, {"lengths": buffer(0x8000000, 2, np.int64)}, hx.InvalidConfiguration, "lengths must be uint32"),
    (attention, {"state_in": view(0x6000000, L([2, 4, 8, 16]), B)}, hx.InvalidConfiguration, "state must be float32"),
    (attention, {"scale": float("inf")}, hx.InvalidConfiguration, "scale must be finite"),
    (attention, {"lengths": buffer(0x8000000, 3, np.uint32)}, hx.LengthMismatch, "2"),
    (attention, {"log_decay": buffer(0x4000000, 2, F)}, hx.LengthMismatch, "4"),
    (attention, {"k": view(0x2000000, L([2, 5, 3, 8]), F), "v": view(0x3000000, L([2, 5, 3, 16]), F)},
     hx.DispatchFailed, "must be a multiple of the key/value heads"),
    (attention, {"v": view(0x3000000, L([2, 5, 4, 16]), F)}, hx.DispatchFailed, "attention value has shape"),
    (attention, {"state_in": view(0x6000000, L([2, 4, 16, 8]), F)}, hx.DispatchFailed, "attention state has shape"),
    (attention, {"q": view(0x1000000, L([2, 5, 32]), F)}, hx.DispatchFailed, "rank"),
    (attention, {"state_out": view(0x7000000, N([2, 4, 8, 16], [0, 128, 16, 1]), F)}, hx.DispatchFailed,
     "reach an element twice"),
    (attention, {"output": view(0x3000000, L([2, 5, 4, 16]), F)}, hx.DispatchFailed, "must not overlap the value"),
    (attention, {"output": view(0x7000040, L([2, 5, 4, 16]), F)}, hx.DispatchFailed,
     "must not overlap the state output"),
    (attention, {"state_out": view(0x6000040, L([2, 4, 8, 16]), F)}, hx.DispatchFailed, "be the view of the state"),
    (attention, {"state_out": view(0x8000000, L([2, 4, 8, 16]), F)}, hx.DispatchFailed,
     "must not overlap the sequence lengths"),
    (attention, {"q": view(0x1000000, L([2, 5, 4, 257]), F), "k": view(0x2000000, L([2, 5, 2, 257]), F),
                 "state_in": None, "state_out": None}, hx.DispatchFailed, "at most 256 wide"),
]


@pytest.mark.parametrize("call,change,error,words", REFUSED, ids=[f"{r[0].__name__}-{i}" for i, r in enumerate(REFUSED)])
def test_refusals(call, change, error, words):
    with pytest.raises(hx.HephaestusError) as e:
        call(**change)
    assert type(e.value) is error and words in str(e.value), e.value


@pytest.mark.parametrize("call", [norm, matmul, attention])
def test_operands_that_pass_reach_the_device(call):
    """The same calls without a fault get as far as the missing device."""
    with pytest.raises(hx.HephaestusError) as e:
        call()
    assert "device" in str(e.value)


@pytest.mark.parametrize("call,change", [
    (norm, {"residual_out": view(0x1000000, L([4, 64]), F)}),
    (norm, {"residual_out": view(0x5000000, L([4, 64]), F)}),
    (norm, {"x": view(0x1000000, N([4, 64], [0, 1]), F, 64)}),
    (attention, {"state_out": view(0x6000000, L([2, 4, 8, 16]), F)}),
    (attention, {"state_in": None, "state_out": None, "lengths": None}),
])
def test_views_in_place_are_taken(call, change):
    with pytest.raises(hx.HephaestusError) as e:
        call(**change)
    assert "device" in str(e.value)


def test_bfloat16_conversions():
    rng = np.random.default_rng(0)
    bits = rng.integers(0, 2**16, 4000, dtype=np.uint16)
    exact = hx.float32_from_bfloat16(bits.view(hx.bfloat16))
    back = hx.bfloat16_from_float32(exact).view(np.uint16)
    same = ~np.isnan(exact)
    assert np.array_equal(back[same], bits[same])
    assert np.isnan(hx.float32_from_bfloat16(back.view(hx.bfloat16))[~same]).all()
    x = np.array([1.0 + 2.0**-8, 1.0 + 3 * 2.0**-8, 1.0 + 2.0**-8 + 2.0**-20, 3.4e38, -0.0, np.nan, -np.inf], np.float32)
    want = np.array([1.0, 1.0 + 2.0**-6, 1.0 + 2.0**-7, np.inf, -0.0, np.nan, -np.inf], np.float32)
    got = hx.float32_from_bfloat16(hx.bfloat16_from_float32(x))
    assert np.array_equal(got, want, equal_nan=True) and np.signbit(got[4])


def test_borrowed_memory():
    device = hx.RocmDevice.__new__(hx.RocmDevice)
    device.handle = None
    owner = np.zeros(4)
    b = device.borrow(0x1000, hx.bfloat16, 8, owner)
    assert (b.ptr, len(b), b.itemsize) == (0x1000, 8, 2) and b.owner is owner
    b.free()
    assert b.ptr is None
    for args in ((0x1000, np.float32, 4, None), (0, np.float32, 4, owner), (0x1000, np.float32, -1, owner)):
        with pytest.raises(hx.InvalidConfiguration):
            device.borrow(*args)


def test_other_operators_refuse_bfloat16():
    x = view(0x1000000, L([4, 64]), B)
    for call in (lambda: hx.RocmFullReductionOps().reduce_full_into(NoDevice, hx.SumOp, x, view(0x2000000, L([1]), B)),
                 lambda: hx.RocmScanOps().inclusive_scan_into(NoDevice, x.buffer, buffer(0x2000000, 256, B)),
                 lambda: hx.RocmAxisReductionOps().reduce_axis_into(
                     NoDevice, hx.SumOp, x, 1, view(0x2000000, L([4, 1]), B))):
        with pytest.raises(hx.InvalidConfiguration, match="unknown dtype"):
            call()
