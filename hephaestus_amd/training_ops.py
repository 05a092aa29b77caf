"""Operators that a scan-type language model is trained with, over the C ABI
(hx_layer_norm, hx_gated_recurrence, hx_linear_cross_entropy and their
*_backward of include/hx.h, which states their formulas and rules).

They have no counterpart in the reference; they follow its conventions like the
layer operators: `*_into` calls run at once on a stream, `prepare_*` calls bind
their operands and return a `PreparedPlan` that allocates nothing when
dispatched.  Every call validates first and leaves the outputs of a refused call
untouched.

Element types are float32 and bfloat16 (`hephaestus_amd.bfloat16`).  The last
dimension of every view is contiguous.
"""
from __future__ import annotations

import numpy as np

from . import _ffi
from .device import RocmBuffer, RocmDevice
from .layer_ops import _element, _prepare, _typed, _vec, _view
from .layout import StridedView
from .ops import PreparedPlan

#: A target that leaves its row out, whatever the vocabulary.
NO_TARGET = 0xFFFFFFFF


def _same(operands, like: StridedView) -> None:
    """Every operand given, a view or a buffer, has the element type of `like`."""
    for operand, what in operands:
        if operand is not None:
            _typed(operand.buffer if isinstance(operand, StridedView) else operand, like.buffer.dtype, what)


def _floats(operands) -> None:
    for operand, what in operands:
        if operand is not None:
            _typed(operand.buffer if isinstance(operand, StridedView) else operand, np.float32, what)


class RocmLayerNormOps:
    """Layer norm of rows with the residual's addition, and its backward pass
    (hx_layer_norm, hx_layer_norm_backward)."""

    @staticmethod
    def _args(x, weight, bias, epsilon, output, residual, residual_out, mean, rstd):
        dtype = _element(x, "norm input")
        _same(((residual, "residual"), (residual_out, "residual output"), (weight, "norm weight"),
               (bias, "norm bias"), (output, "norm output")), x)
        _floats(((mean, "norm mean"), (rstd, "norm rstd")))
        return (dtype, *_view(x), *_view(residual), *_vec(weight), *_vec(bias), float(epsilon), *_view(residual_out),
                *_view(output), *_vec(mean), *_vec(rstd))

    def layer_norm_into(self, device: RocmDevice, x: StridedView, weight: RocmBuffer, bias: RocmBuffer | None,
                        epsilon: float, output: StridedView, residual: StridedView | None = None,
                        residual_out: StridedView | None = None, mean: RocmBuffer | None = None,
                        rstd: RocmBuffer | None = None, stream=None) -> None:
        args = self._args(x, weight, bias, epsilon, output, residual, residual_out, mean, rstd)
        _ffi.check(_ffi.lib().hx_layer_norm(device.handle, *args, stream))

    def prepare_layer_norm(self, device: RocmDevice, x: StridedView, weight: RocmBuffer, bias: RocmBuffer | None,
                           epsilon: float, output: StridedView, residual: StridedView | None = None,
                           residual_out: StridedView | None = None, mean: RocmBuffer | None = None,
                           rstd: RocmBuffer | None = None) -> PreparedPlan:
        args = self._args(x, weight, bias, epsilon, output, residual, residual_out, mean, rstd)
        return _prepare(device, _ffi.lib().hx_prepare_layer_norm, args,
                        (x, weight, bias, output, residual, residual_out, mean, rstd))

    @staticmethod
    def _backward_args(grad_out, x, weight, mean, rstd, grad_in, residual_grad, grad_weight, grad_bias):
        dtype = _element(x, "norm input")
        _same(((grad_out, "gradient of the norm output"), (weight, "norm weight"), (grad_in, "gradient of the norm input"),
               (residual_grad, "gradient past the norm")), x)
        _floats(((mean, "norm mean"), (rstd, "norm rstd"), (grad_weight, "gradient of the norm weight"),
                 (grad_bias, "gradient of the norm bias")))
        return (dtype, *_view(grad_out), *_view(x), *_vec(weight), *_vec(mean), *_vec(rstd), *_view(residual_grad),
                *_view(grad_in), *_vec(grad_weight), *_vec(grad_bias))

    def layer_norm_backward_into(self, device: RocmDevice, grad_out: StridedView, x: StridedView, weight: RocmBuffer,
                                 mean: RocmBuffer, rstd: RocmBuffer, grad_in: StridedView,
                                 residual_grad: StridedView | None = None, grad_weight: RocmBuffer | None = None,
                                 grad_bias: RocmBuffer | None = None, stream=None) -> None:
        args = self._backward_args(grad_out, x, weight, mean, rstd, grad_in, residual_grad, grad_weight, grad_bias)
        _ffi.check(_ffi.lib().hx_layer_norm_backward(device.handle, *args, stream))

    def prepare_layer_norm_backward(self, device: RocmDevice, grad_out: StridedView, x: StridedView,
                                    weight: RocmBuffer, mean: RocmBuffer, rstd: RocmBuffer, grad_in: StridedView,
                                    residual_grad: StridedView | None = None, grad_weight: RocmBuffer | None = None,
                                    grad_bias: RocmBuffer | None = None) -> PreparedPlan:
        args = self._backward_args(grad_out, x, weight, mean, rstd, grad_in, residual_grad, grad_weight, grad_bias)
        return _prepare(device, _ffi.lib().hx_prepare_layer_norm_backward, args,
                        (grad_out, x, weight, mean, rstd, grad_in, residual_grad, grad_weight, grad_bias))


class RocmRecurrenceOps:
    """Gated recurrence of each channel along the tokens, h_t = f_t·h_{t-1} +
    (1 - f_t)·x_t with f the gate's sigmoid, and its backward pass
    (hx_gated_recurrence, hx_gated_recurrence_backward)."""

    @staticmethod
    def _args(gate, x, output, state_in, state_out, lengths):
        dtype = _element(x, "recurrence input")
        _same(((gate, "recurrence gate"), (output, "recurrence output")), x)
        _floats(((state_in, "recurrence state"), (state_out, "recurrence state output")))
        if lengths is not None:
            _typed(lengths, np.uint32, "sequence lengths")
        return (dtype, *_view(gate), *_view(x), *_view(state_in), *_vec(lengths), *_view(output), *_view(state_out))

    def gated_recurrence_into(self, device: RocmDevice, gate: StridedView, x: StridedView, output: StridedView,
                              state_in: StridedView | None = None, state_out: StridedView | None = None,
                              lengths: RocmBuffer | None = None, stream=None) -> None:
        args = self._args(gate, x, output, state_in, state_out, lengths)
        _ffi.check(_ffi.lib().hx_gated_recurrence(device.handle, *args, stream))

    def prepare_gated_recurrence(self, device: RocmDevice, gate: StridedView, x: StridedView, output: StridedView,
                                 state_in: StridedView | None = None, state_out: StridedView | None = None,
                                 lengths: RocmBuffer | None = None) -> PreparedPlan:
        args = self._args(gate, x, output, state_in, state_out, lengths)
        return _prepare(device, _ffi.lib().hx_prepare_gated_recurrence, args,
                        (gate, x, output, state_in, state_out, lengths))

    @staticmethod
    def _backward_args(gate, x, h, grad_out, grad_gate, grad_x, state_in, grad_state_out, grad_state_in, lengths):
        dtype = _element(x, "recurrence input")
        _same(((gate, "recurrence gate"), (h, "recurrence output"), (grad_out, "gradient of the recurrence output"),
               (grad_gate, "gradient of the gate"), (grad_x, "gradient of the recurrence input")), x)
        _floats(((state_in, "recurrence state"), (grad_state_out, "gradient of the state output"),
                 (grad_state_in, "gradient of the state")))
        if lengths is not None:
            _typed(lengths, np.uint32, "sequence lengths")
        return (dtype, *_view(gate), *_view(x), *_view(h), *_view(state_in), *_vec(lengths), *_view(grad_out),
                *_view(grad_state_out), *_view(grad_gate), *_view(grad_x), *_view(grad_state_in))

    def gated_recurrence_backward_into(self, device: RocmDevice, gate: StridedView, x: StridedView, h: StridedView,
                                       grad_out: StridedView, grad_gate: StridedView, grad_x: StridedView,
                                       state_in: StridedView | None = None, grad_state_out: StridedView | None = None,
                                       grad_state_in: StridedView | None = None, lengths: RocmBuffer | None = None,
                                       stream=None) -> None:
        args = self._backward_args(gate, x, h, grad_out, grad_gate, grad_x, state_in, grad_state_out, grad_state_in,
                                   lengths)
        _ffi.check(_ffi.lib().hx_gated_recurrence_backward(device.handle, *args, stream))

    def prepare_gated_recurrence_backward(self, device: RocmDevice, gate: StridedView, x: StridedView, h: StridedView,
                                          grad_out: StridedView, grad_gate: StridedView, grad_x: StridedView,
                                          state_in: StridedView | None = None,
                                          grad_state_out: StridedView | None = None,
                                          grad_state_in: StridedView | None = None,
                                          lengths: RocmBuffer | None = None) -> PreparedPlan:
        args = self._backward_args(gate, x, h, grad_out, grad_gate, grad_x, state_in, grad_state_out, grad_state_in,
                                   lengths)
        return _prepare(device, _ffi.lib().hx_prepare_gated_recurrence_backward, args,
                        (gate, x, h, grad_out, grad_gate, grad_x, state_in, grad_state_out, grad_state_in, lengths))


class RocmLossOps:
    """Softmax cross entropy of the logits x·weightᵀ over a vocabulary, which are
    not kept, and its backward pass (hx_linear_cross_entropy,
    hx_linear_cross_entropy_backward).  A target not below the vocabulary, such as
    `NO_TARGET`, leaves its row out."""

    @staticmethod
    def _args(x, weight, targets, loss, lse):
        dtype = _element(x, "loss input")
        _same(((weight, "vocabulary weight"),), x)
        _typed(targets, np.uint32, "targets")
        _floats(((loss, "loss"), (lse, "logarithms of the denominators")))
        return dtype, *_view(x), *_view(weight), *_vec(targets), *_vec(loss), *_vec(lse)

    def linear_cross_entropy_into(self, device: RocmDevice, x: StridedView, weight: StridedView, targets: RocmBuffer,
                                  loss: RocmBuffer, lse: RocmBuffer | None = None, stream=None) -> None:
        args = self._args(x, weight, targets, loss, lse)
        _ffi.check(_ffi.lib().hx_linear_cross_entropy(device.handle, *args, stream))

    def prepare_linear_cross_entropy(self, device: RocmDevice, x: StridedView, weight: StridedView,
                                     targets: RocmBuffer, loss: RocmBuffer,
                                     lse: RocmBuffer | None = None) -> PreparedPlan:
        args = self._args(x, weight, targets, loss, lse)
        return _prepare(device, _ffi.lib().hx_prepare_linear_cross_entropy, args, (x, weight, targets, loss, lse))

    @staticmethod
    def _backward_args(x, weight, targets, lse, grad, grad_x, grad_weight):
        dtype = _element(x, "loss input")
        _same(((weight, "vocabulary weight"), (grad_x, "gradient of the loss input"),
               (grad_weight, "gradient of the vocabulary weight")), x)
        _typed(targets, np.uint32, "targets")
        _floats(((lse, "logarithms of the denominators"), (grad, "gradient of the loss")))
        return (dtype, *_view(x), *_view(weight), *_vec(targets), *_vec(lse), *_vec(grad), *_view(grad_x),
                *_view(grad_weight))

    def linear_cross_entropy_backward_into(self, device: RocmDevice, x: StridedView, weight: StridedView,
                                           targets: RocmBuffer, lse: RocmBuffer, grad: RocmBuffer,
                                           grad_x: StridedView | None = None, grad_weight: StridedView | None = None,
                                           stream=None) -> None:
        args = self._backward_args(x, weight, targets, lse, grad, grad_x, grad_weight)
        _ffi.check(_ffi.lib().hx_linear_cross_entropy_backward(device.handle, *args, stream))

    def prepare_linear_cross_entropy_backward(self, device: RocmDevice, x: StridedView, weight: StridedView,
                                              targets: RocmBuffer, lse: RocmBuffer, grad: RocmBuffer,
                                              grad_x: StridedView | None = None,
                                              grad_weight: StridedView | None = None) -> PreparedPlan:
        args = self._backward_args(x, weight, targets, lse, grad, grad_x, grad_weight)
        return _prepare(device, _ffi.lib().hx_prepare_linear_cross_entropy_backward, args,
                        (x, weight, targets, lse, grad, grad_x, grad_weight))
