"""Recurrences of more channels than the blocks of a launch hold."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from hephaestus_amd import Layout, StridedView
from layer_reference import rounded
from training_reference import gated_recurrence, gated_recurrence_backward, near

pytestmark = pytest.mark.gpu


# A launch has 2^28 channels of f32, and of bf16 off dwords, 2^29 of bf16.
@pytest.mark.parametrize("t,run", [(np.float32, 1 << 28), (hx.bfloat16, 1 << 29), (hx.bfloat16, 1 << 28)])
def test_channels_of_two_launches(device, t, run):
    """Zeros but for the channels around the launches' ends."""
    channels = run + (431 if t == np.float32 or run == 1 << 28 else 430)
    looked_at = [0, run - 200, run, channels - 200]  # apart from each other
    rng = np.random.default_rng(3)

    def operand(dtype, values):
        buffer = device.alloc_zeroed(dtype, channels)
        for i, at in enumerate(looked_at):
            device.write_sub_buffer(buffer, at, values[i])
        return buffer

    def read(buffer):
        return np.stack([device.download_owned(device.borrow(buffer.ptr + at * buffer.itemsize, buffer.dtype, 200, buffer))
                         for at in looked_at])

    def tokens(buffer):
        return StridedView(buffer, Layout.c_contiguous([1, 1, channels]))

    def state(buffer):
        return StridedView(buffer, Layout.c_contiguous([1, channels]))

    gate, x, dy = (rounded(rng.normal(size=(4, 200)), t) for _ in range(3))
    first, dlast = rng.normal(size=(2, 4, 200)).astype(np.float32)
    at = {"gate": operand(t, gate), "x": operand(t, x), "first": operand(np.float32, first)}
    h, last = device.alloc_uninitialized(t, channels), device.alloc_uninitialized(np.float32, channels)
    ops = hx.RocmRecurrenceOps()
    ops.gated_recurrence_into(device, tokens(at["gate"]), tokens(at["x"]), tokens(h), state_in=state(at["first"]),
                              state_out=state(last))
    device.synchronize()
    value, bound = gated_recurrence(gate[:, None], x[:, None], first)
    got = {"h": read(h), "last": read(last)}
    near(got["h"], value["h"][:, 0], bound["h"][:, 0], "h")
    near(got["last"], value["last"], bound["last"], "last")
    at["dy"], at["dlast"] = operand(t, dy), operand(np.float32, dlast)
    dgate, dx = device.alloc_uninitialized(t, channels), device.alloc_uninitialized(t, channels)
    ops.gated_recurrence_backward_into(device, tokens(at["gate"]), tokens(at["x"]), tokens(h), tokens(at["dy"]), tokens(dgate),
                                       tokens(dx), state_in=state(at["first"]), grad_state_out=state(at["dlast"]),
                                       grad_state_in=state(last))
    device.synchronize()
    value, bound = gated_recurrence_backward(gate[:, None], x[:, None], got["h"][:, None], dy[:, None], first, dlast)
    near(read(dgate), value["dgate"][:, 0], bound["dgate"][:, 0], "dgate")
    near(read(dx), value["dx"][:, 0], bound["dx"][:, 0], "dx")
    near(read(last), value["dfirst"], bound["dfirst"], "dfirst")


def test_plan_of_three_launches(device):
    """2^29 + 64 channels of f32: with 512 threads a block one launch would pass 2^32."""
    channels = (1 << 29) + 64
    gate, x = device.alloc_zeroed(np.float32, channels), device.alloc_zeroed(np.float32, channels)
    ends = np.arange(1, 65, dtype=np.float32)
    device.write_sub_buffer(x, channels - 64, ends)
    out = device.alloc_uninitialized(np.float32, channels)
    views = [StridedView(b, Layout.c_contiguous([1, 1, channels])) for b in (gate, x, out)]
    plan = hx.RocmRecurrenceOps().prepare_gated_recurrence(device, *views)
    plan.dispatch()
    device.synchronize()
    got = device.download_owned(device.borrow(out.ptr + 4 * (channels - 128), np.float32, 128, out))
    assert np.array_equal(got, np.concatenate([np.zeros(64, np.float32), ends / 2]))
