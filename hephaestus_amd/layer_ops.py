"""Operators of a linear-attention layer served in 8 bits, over the C ABI
(hx_rms_norm_quantize, hx_matmul_i8, hx_linear_attention of include/hx.h,
which states their formulas and rules).

They have no counterpart in the reference; they follow its conventions:
`*_into` calls run at once on a stream, `prepare_*` calls bind their operands
and return a `PreparedPlan` that allocates nothing when dispatched.  Every call
validates first and leaves the outputs of a refused call untouched.

Element types are float32 and bfloat16 (`hephaestus_amd.bfloat16`), int8 for
what is quantised.  The last dimension of every view is contiguous.
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import _ffi, errors
from .device import RocmBuffer, RocmDevice, bfloat16, hx_dtype
from .layout import StridedView
from .ops import PreparedPlan


def _element(view: StridedView, what: str) -> int:
    """The hx_dtype of a float32 or bfloat16 operand."""
    if view.buffer.dtype not in (np.dtype(np.float32), bfloat16):
        raise errors.InvalidConfiguration(f"{what} must be float32 or bfloat16, got {view.buffer.dtype}")
    return hx_dtype(view.buffer.dtype)


def _typed(buffer: RocmBuffer, dtype, what: str) -> None:
    if buffer.dtype != np.dtype(dtype):
        raise errors.InvalidConfiguration(f"{what} must be {np.dtype(dtype)}, got {buffer.dtype}")


def _vec(buffer: RocmBuffer | None):
    """A whole buffer as (pointer, length)."""
    return (None, 0) if buffer is None else (buffer.ptr, len(buffer))


def _view(view: StridedView | None):
    """A view as (pointer, buffer length, layout)."""
    if view is None:
        return None, 0, None
    return view.buffer.ptr, len(view.buffer), ctypes.byref(_ffi.layout_struct(view.layout))


def _prepare(device: RocmDevice, fn, args: tuple, keep: tuple) -> PreparedPlan:
    plan = ctypes.c_void_p()
    _ffi.check(fn(device.handle, *args, ctypes.byref(plan)))
    return PreparedPlan(device, plan.value, keep)


class RocmNormOps:
    """RMS norm of rows with the residual's addition, quantised to 8 bits with
    a scale for each row (hx_rms_norm_quantize)."""

    @staticmethod
    def _args(x, weight, epsilon, quantized, scales, residual, residual_out):
        dtype = _element(x, "norm input")
        for view, what in ((residual, "residual"), (residual_out, "residual output")):
            if view is not None:
                _typed(view.buffer, x.buffer.dtype, what)
        _typed(weight, x.buffer.dtype, "norm weight")
        _typed(quantized.buffer, np.int8, "quantized output")
        _typed(scales, np.float32, "quantized scales")
        return (dtype, *_view(x), *_view(residual), *_vec(weight), float(epsilon), *_view(residual_out),
                *_view(quantized), *_vec(scales))

    def rms_norm_quantize_into(self, device: RocmDevice, x: StridedView, weight: RocmBuffer, epsilon: float,
                               quantized: StridedView, scales: RocmBuffer, residual: StridedView | None = None,
                               residual_out: StridedView | None = None, stream=None) -> None:
        args = self._args(x, weight, epsilon, quantized, scales, residual, residual_out)
        _ffi.check(_ffi.lib().hx_rms_norm_quantize(device.handle, *args, stream))

    def prepare_rms_norm_quantize(self, device: RocmDevice, x: StridedView, weight: RocmBuffer, epsilon: float,
                                  quantized: StridedView, scales: RocmBuffer, residual: StridedView | None = None,
                                  residual_out: StridedView | None = None) -> PreparedPlan:
        args = self._args(x, weight, epsilon, quantized, scales, residual, residual_out)
        return _prepare(device, _ffi.lib().hx_prepare_rms_norm_quantize, args,
                        (x, weight, quantized, scales, residual, residual_out))


class RocmMatrixOps:
    """Products of 8-bit integers with a scale for each token (row of a) and
    channel (row of b), in float32 or bfloat16 (hx_matmul_i8)."""

    @staticmethod
    def _args(a, a_scales, b, b_scales, output):
        for view, scales, what in ((a, a_scales, "a"), (b, b_scales, "b")):
            _typed(view.buffer, np.int8, f"matmul operand {what}")
            _typed(scales, np.float32, f"matmul scales of {what}")
        dtype = _element(output, "matmul output")
        return (*_view(a), *_vec(a_scales), *_view(b), *_vec(b_scales), dtype, *_view(output))

    def matmul_i8_into(self, device: RocmDevice, a: StridedView, a_scales: RocmBuffer, b: StridedView,
                       b_scales: RocmBuffer, output: StridedView, stream=None) -> None:
        args = self._args(a, a_scales, b, b_scales, output)
        _ffi.check(_ffi.lib().hx_matmul_i8(device.handle, *args, stream))

    def prepare_matmul_i8(self, device: RocmDevice, a: StridedView, a_scales: RocmBuffer, b: StridedView,
                          b_scales: RocmBuffer, output: StridedView) -> PreparedPlan:
        args = self._args(a, a_scales, b, b_scales, output)
        return _prepare(device, _ffi.lib().hx_prepare_matmul_i8, args, (a, a_scales, b, b_scales, output))


class RocmLinearAttentionOps:
    """Linear attention with a decay for each head: S_t = e^g·S_{t-1} + k_tᵀv_t,
    o_t = scale·q_t·S_t (hx_linear_attention).  `scale` defaults to 1/√dk."""

    @staticmethod
    def _args(q, k, v, log_decay, output, scale, state_in, state_out, lengths):
        dtype = _element(q, "attention query")
        for view, what in ((k, "attention key"), (v, "attention value"), (output, "attention output")):
            _typed(view.buffer, q.buffer.dtype, what)
        _typed(log_decay, np.float32, "log decay")
        for view, what in ((state_in, "attention state"), (state_out, "attention state output")):
            if view is not None:
                _typed(view.buffer, np.float32, what)
        if lengths is not None:
            _typed(lengths, np.uint32, "sequence lengths")
        if scale is None:
            scale = max(1, q.layout.shape[-1]) ** -0.5
        return (dtype, *_view(q), *_view(k), *_view(v), *_vec(log_decay), float(scale), *_view(state_in),
                *_view(state_out), *_vec(lengths), *_view(output))

    def linear_attention_into(self, device: RocmDevice, q: StridedView, k: StridedView, v: StridedView,
                              log_decay: RocmBuffer, output: StridedView, scale: float | None = None,
                              state_in: StridedView | None = None, state_out: StridedView | None = None,
                              lengths: RocmBuffer | None = None, stream=None) -> None:
        args = self._args(q, k, v, log_decay, output, scale, state_in, state_out, lengths)
        _ffi.check(_ffi.lib().hx_linear_attention(device.handle, *args, stream))

    def prepare_linear_attention(self, device: RocmDevice, q: StridedView, k: StridedView, v: StridedView,
                                 log_decay: RocmBuffer, output: StridedView, scale: float | None = None,
                                 state_in: StridedView | None = None, state_out: StridedView | None = None,
                                 lengths: RocmBuffer | None = None) -> PreparedPlan:
        args = self._args(q, k, v, log_decay, output, scale, state_in, state_out, lengths)
        return _prepare(device, _ffi.lib().hx_prepare_linear_attention, args,
                        (q, k, v, log_decay, output, state_in, state_out, lengths))
