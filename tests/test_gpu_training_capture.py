"""Which immediate training operators a stream under capture takes: those without
scratch are recorded and replay, the others refuse before anything is queued."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from layer_reference import padded, rounded, vector
from test_gpu_gated_recurrence import operands as recurrence_operands
from test_gpu_layer_norm import operands as norm_operands, stats_of
from test_gpu_training_streams import Capture, Stream
from training_reference import TYPES, gated_recurrence_backward, layer_norm_backward, near

pytestmark = pytest.mark.gpu


def norm_backward(device, t, with_sums):
    x, _, w, _, dy, past = norm_operands(t, 37, 300, 1)
    mean, rstd = stats_of(x)
    vd, read = padded(device, rounded(np.full(x.shape, 7.0), t))
    sums = {"grad_weight": vector(device, np.zeros(300, np.float32))} if with_sums else {}
    args = (padded(device, dy)[0], padded(device, x)[0], vector(device, w), vector(device, mean), vector(device, rstd), vd)
    vp = padded(device, past)[0]

    def call(stream):
        hx.RocmLayerNormOps().layer_norm_backward_into(device, *args, residual_grad=vp, **sums, stream=stream)

    def check():
        value, bound = layer_norm_backward(dy, x, w, mean, rstd, past)
        near(read(), value["dh"], bound["dh"], "dh")

    return call, check


def recurrence_backward(device, t, tokens):
    gate, x, dy, first, dlast = recurrence_operands(t, 2, tokens, 70, 2)
    h = rounded(np.random.default_rng(3).normal(size=x.shape), t)
    vz, read_z = padded(device, rounded(np.full(x.shape, 9.0), t))
    vx, read_x = padded(device, rounded(np.full(x.shape, 9.0), t))
    views = [padded(device, v)[0] for v in (gate, x, h, dy)]
    states = {"state_in": padded(device, first)[0], "grad_state_out": padded(device, dlast)[0]}

    def call(stream):
        hx.RocmRecurrenceOps().gated_recurrence_backward_into(device, *views, vz, vx, **states, stream=stream)

    def check():
        value, bound = gated_recurrence_backward(gate, x, h, dy, first, dlast)
        near(read_z(), value["dgate"], bound["dgate"], "dgate")
        near(read_x(), value["dx"], bound["dx"], "dx")

    return call, check


@pytest.mark.parametrize("dtype", TYPES)
def test_calls_without_scratch_are_captured(device, dtype):
    t = TYPES[dtype]
    cases = [norm_backward(device, t, False), recurrence_backward(device, t, 1), recurrence_backward(device, t, 32)]
    stream = Stream()
    capture = Capture(stream)
    try:
        with capture:
            for call, _ in cases:
                call(stream.value)
        for _ in range(3):
            capture.replay()
            for _, check in cases:
                check()
            for call, _ in cases:  # eager calls between the replays
                call(None)
            device.synchronize()
    finally:
        capture.destroy()
        stream.close(device)


@pytest.mark.parametrize("dtype", TYPES)
def test_calls_with_scratch_are_refused(device, dtype):
    t = TYPES[dtype]
    cases = [norm_backward(device, t, True), recurrence_backward(device, t, 700)]
    taken, _ = norm_backward(device, t, False)
    stream = Stream()
    capture = Capture(stream)
    try:
        with capture:
            taken(stream.value)
            for call, _ in cases:
                with pytest.raises(hx.DispatchFailed):
                    call(stream.value)
    finally:
        capture.destroy()
        stream.close(device)
    for call, check in cases:  # and run as ever afterwards
        call(None)
        device.synchronize()
        check()
