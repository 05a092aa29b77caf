"""Operands of the training operators that share one layout object, as callers of the
C ABI and of the C++ interface pass them for views of one shape: what may overlap goes
by which operand it is, not by its layout.  Checks run before a device is touched."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import hephaestus_amd as hx
from hephaestus_amd import Layout, _ffi
from test_layer_refusals import NoDevice

F32 = 0
SHAPES = {"norm": [4, 64], "norm_grad": [4, 64], "scan": [2, 5, 8], "scan_grad": [2, 5, 8], "loss_grad": [6, 6]}
STATE = [2, 8]


def place(i):
    return 0x10000000 * (i + 1)


def call(op, **at):
    """The call with each view at a place of its own, or where `at` says, all views of a
    shape with one layout."""
    names = iter(range(100))
    rows = _ffi.layout_struct(Layout.c_contiguous(SHAPES[op]))
    states = _ffi.layout_struct(Layout.c_contiguous(STATE))
    size, state_size = int(np.prod(SHAPES[op])), int(np.prod(STATE))

    def spot(name):
        own = place(next(names))
        return place(at[name]) if name in at else own

    def view(name):
        return spot(name), size, ctypes.byref(rows)

    def state(name):
        return spot(name), state_size, ctypes.byref(states)

    def vec(name, n):
        return spot(name), n

    lib, none = _ffi.lib(), (None, 0)
    if op == "norm":
        args = (F32, *view("x"), *view("residual"), *vec("weight", 64), *none, 1e-5, *view("residual_out"), *view("out"),
                *none, *none)
        fn = lib.hx_layer_norm
    elif op == "norm_grad":
        args = (F32, *view("grad_out"), *view("x"), *vec("weight", 64), *vec("mean", 4), *vec("rstd", 4),
                *view("residual_grad"), *view("grad_in"), *none, *none)
        fn = lib.hx_layer_norm_backward
    elif op == "scan":
        args = (F32, *view("gate"), *view("x"), *state("state_in"), *none, *view("out"), *state("state_out"))
        fn = lib.hx_gated_recurrence
    elif op == "scan_grad":
        args = (F32, *view("gate"), *view("x"), *view("h"), *state("state_in"), *none, *view("grad_out"),
                *state("grad_state_out"), *view("grad_gate"), *view("grad_x"), *state("grad_state_in"))
        fn = lib.hx_gated_recurrence_backward
    else:
        args = (F32, *view("x"), *view("weight"), *vec("targets", 6), *vec("lse", 6), *vec("grad", 6), *view("grad_x"),
                *view("grad_weight"))
        fn = lib.hx_linear_cross_entropy_backward
    _ffi.check(fn(NoDevice.handle, *args, None))


# Places by the order in which the calls above name their operands.
NORM = {"x": 0, "residual": 1, "weight": 2, "residual_out": 3, "out": 4}
NORM_GRAD = {"grad_out": 0, "x": 1, "weight": 2, "mean": 3, "rstd": 4, "residual_grad": 5, "grad_in": 6}
SCAN = {"gate": 0, "x": 1, "state_in": 2, "out": 3, "state_out": 4}
SCAN_GRAD = {"gate": 0, "x": 1, "h": 2, "state_in": 3, "grad_out": 4, "grad_state_out": 5, "grad_gate": 6, "grad_x": 7,
             "grad_state_in": 8}

REFUSED = [
    ("norm", {"out": NORM["residual_out"]}, "norm output"), ("norm", {"out": NORM["x"]}, "norm output"),
    ("norm", {"out": NORM["residual"]}, "norm output"), ("norm", {"residual_out": NORM["x"], "out": NORM["x"]}, "norm output"),
    ("norm", {"residual_out": NORM["weight"]}, "residual output"),
    ("norm_grad", {"grad_in": NORM_GRAD["x"]}, "gradient of the norm input"),
    ("norm_grad", {"grad_in": NORM_GRAD["weight"]}, "gradient of the norm input"),
    ("scan", {"out": SCAN["x"]}, "recurrence output"), ("scan", {"out": SCAN["gate"]}, "recurrence output"),
    ("scan", {"state_out": SCAN["out"]}, "must not overlap"),
    ("scan_grad", {"grad_gate": SCAN_GRAD["gate"]}, "gradient of the gate"),
    ("scan_grad", {"grad_x": SCAN_GRAD["grad_gate"]}, "must not overlap"),
    ("scan_grad", {"grad_x": SCAN_GRAD["grad_out"]}, "gradient of the recurrence input"),
    ("scan_grad", {"grad_state_in": SCAN_GRAD["state_in"]}, "gradient of the state"),
    ("scan_grad", {"grad_state_in": SCAN_GRAD["grad_state_out"]}, "gradient of the state"),
    ("loss_grad", {"grad_x": 0}, "loss input"), ("loss_grad", {"grad_weight": 1}, "vocabulary weight"),
    ("loss_grad", {"grad_weight": 5}, "must not overlap"),
]
IN_PLACE = [
    ("norm", {}), ("norm", {"residual_out": NORM["x"]}), ("norm", {"residual_out": NORM["residual"]}),
    ("norm", {"residual_out": NORM["x"], "residual": NORM["x"]}), ("norm_grad", {}),
    ("norm_grad", {"grad_in": NORM_GRAD["grad_out"]}), ("norm_grad", {"grad_in": NORM_GRAD["residual_grad"]}),
    ("norm_grad", {"grad_in": NORM_GRAD["grad_out"], "residual_grad": NORM_GRAD["grad_out"]}),
    ("scan", {}), ("scan", {"state_out": SCAN["state_in"]}), ("scan_grad", {}), ("loss_grad", {}),
]


@pytest.mark.parametrize("op,at,what", REFUSED)
def test_overlaps_are_refused(op, at, what):
    with pytest.raises(hx.DispatchFailed, match="must not overlap") as refused:
        call(op, **at)
    assert what in str(refused.value)


@pytest.mark.parametrize("op,at", IN_PLACE)
def test_what_may_be_in_place_is_taken(op, at):
    """The checks pass: what is then missing is the device."""
    with pytest.raises(hx.HephaestusError, match="null device"):
        call(op, **at)
