"""What the training operators refuse, and in which words.  Checks run before a
device is touched, so these need none (the calls go to a device that was never
opened)."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
from hephaestus_amd import Layout, RocmBuffer, StridedView
from test_layer_refusals import NoDevice, buffer, view

L, N = Layout.c_contiguous, Layout.try_new
F, B, U = np.float32, hx.bfloat16, np.uint32


def place(i):
    return 0x10000000 * (i + 1)


def call(method, **defaults):
    def run(**change):
        getattr(defaults["ops"], method)(NoDevice, **{k: v for k, v in {**defaults, **change}.items() if k != "ops"})

    run.defaults = defaults
    run.method = method
    return run


norm = call("layer_norm_into", ops=hx.RocmLayerNormOps(), x=view(place(0), L([4, 64]), F), weight=buffer(place(1), 64, F),
            bias=buffer(place(2), 64, F), epsilon=1e-5, output=view(place(3), L([4, 64]), F),
            residual=view(place(4), L([4, 64]), F), residual_out=view(place(5), L([4, 64]), F),
            mean=buffer(place(6), 4, F), rstd=buffer(place(7), 4, F))
norm_grad = call("layer_norm_backward_into", ops=hx.RocmLayerNormOps(), grad_out=view(place(0), L([4, 64]), F),
                 x=view(place(1), L([4, 64]), F), weight=buffer(place(2), 64, F), mean=buffer(place(3), 4, F),
                 rstd=buffer(place(4), 4, F), grad_in=view(place(5), L([4, 64]), F),
                 residual_grad=view(place(6), L([4, 64]), F), grad_weight=buffer(place(7), 64, F),
                 grad_bias=buffer(place(8), 64, F))
scan = call("gated_recurrence_into", ops=hx.RocmRecurrenceOps(), gate=view(place(0), L([2, 5, 8]), F),
            x=view(place(1), L([2, 5, 8]), F), output=view(place(2), L([2, 5, 8]), F),
            state_in=view(place(3), L([2, 8]), F), state_out=view(place(4), L([2, 8]), F), lengths=buffer(place(5), 2, U))
scan_grad = call("gated_recurrence_backward_into", ops=hx.RocmRecurrenceOps(), gate=view(place(0), L([2, 5, 8]), F),
                 x=view(place(1), L([2, 5, 8]), F), h=view(place(2), L([2, 5, 8]), F),
                 grad_out=view(place(3), L([2, 5, 8]), F), grad_gate=view(place(4), L([2, 5, 8]), F),
                 grad_x=view(place(5), L([2, 5, 8]), F), state_in=view(place(6), L([2, 8]), F),
                 grad_state_out=view(place(7), L([2, 8]), F), grad_state_in=view(place(8), L([2, 8]), F),
                 lengths=buffer(place(9), 2, U))
loss = call("linear_cross_entropy_into", ops=hx.RocmLossOps(), x=view(place(0), L([4, 8]), F),
            weight=view(place(1), L([9, 8]), F), targets=buffer(place(2), 4, U), loss=buffer(place(3), 4, F),
            lse=buffer(place(4), 4, F))
loss_grad = call("linear_cross_entropy_backward_into", ops=hx.RocmLossOps(), x=view(place(0), L([4, 8]), F),
                 weight=view(place(1), L([9, 8]), F), targets=buffer(place(2), 4, U), lse=buffer(place(3), 4, F),
                 grad=buffer(place(4), 4, F), grad_x=view(place(5), L([4, 8]), F),
                 grad_weight=view(place(6), L([9, 8]), F))

IC, DF, LM = hx.InvalidConfiguration, hx.DispatchFailed, hx.LengthMismatch
REFUSED = [
    # norm
    (norm, {"x": view(place(0), L([4, 64]), np.int32)}, IC, "float32 or bfloat16"),
    (norm, {"weight": buffer(place(1), 64, B)}, IC, "norm weight must be float32"),
    (norm, {"bias": buffer(place(2), 64, B)}, IC, "norm bias must be float32"),
    (norm, {"output": view(place(3), L([4, 64]), B)}, IC, "norm output must be float32"),
    (norm, {"mean": buffer(place(6), 4, B)}, IC, "norm mean must be float32"),
    (norm, {"epsilon": -1.0}, IC, "epsilon"),
    (norm, {"epsilon": float("nan")}, IC, "epsilon"),
    (norm, {"weight": buffer(place(1), 63, F)}, LM, "64"),
    (norm, {"bias": buffer(place(2), 65, F)}, LM, "64"),
    (norm, {"rstd": buffer(place(7), 5, F)}, LM, "4"),
    (norm, {"x": view(place(0), L([256]), F)}, DF, "rank-2"),
    (norm, {"residual": view(place(4), L([4, 63]), F)}, DF, "residual has shape"),
    (norm, {"output": view(place(3), L([3, 64]), F)}, DF, "norm output has shape"),
    (norm, {"x": view(place(0), N([4, 64], [128, 2]), F, 512)}, DF, "contiguous last dimension"),
    (norm, {"x": view(place(0), L([4, 64]), F, 255)}, DF, "layout rejected"),
    (norm, {"x": view(0, L([4, 64]), F)}, DF, "null"),
    (norm, {"x": view(place(0) + 2, L([4, 64]), F)}, DF, "not aligned"),
    (norm, {"mean": buffer(place(6) + 2, 4, F)}, DF, "not aligned"),
    (norm, {"output": view(place(3), N([4, 64], [0, 1]), F)}, DF, "reach an element twice"),
    (norm, {"output": view(place(0), L([4, 64]), F)}, DF, "norm output must not overlap norm input"),
    (norm, {"output": view(place(5), L([4, 64]), F)}, DF, "must not overlap"),
    (norm, {"mean": buffer(place(7), 4, F)}, DF, "must not overlap"),
    (norm, {"residual_out": view(place(0) + 256, L([4, 64]), F)}, DF, "must be the view of norm input or not overlap it"),
    # norm, backward
    (norm_grad, {"grad_out": view(place(0), L([4, 64]), B)}, IC, "gradient of the norm output must be float32"),
    (norm_grad, {"grad_weight": buffer(place(7), 64, B)}, IC, "gradient of the norm weight must be float32"),
    (norm_grad, {"mean": buffer(place(3), 5, F)}, LM, "4"),
    (norm_grad, {"grad_bias": buffer(place(8), 63, F)}, LM, "64"),
    (norm_grad, {"grad_in": view(place(5), L([4, 32]), F)}, DF, "gradient of the norm input has shape"),
    (norm_grad, {"grad_in": view(place(1), L([4, 64]), F)}, DF, "must not overlap norm input"),
    (norm_grad, {"grad_in": view(place(0) + 4, L([4, 64]), F)}, DF, "must be the view of gradient of the norm output"),
    (norm_grad, {"grad_in": view(place(6), N([4, 64], [-64, 1], 192), F)}, DF, "must be the view of gradient past the norm"),
    (norm_grad, {"grad_weight": buffer(place(8) + 64, 64, F)}, DF, "must not overlap"),
    (norm_grad, {"grad_weight": buffer(place(5) + 64, 64, F)}, DF, "must not overlap"),
    (norm_grad, {k: view(place(i), L([1, 65535 * 1024 + 1]), F) for i, k in enumerate(("grad_out", "x", "grad_in"))} | {
        "weight": buffer(place(12), 65535 * 1024 + 1, F), "mean": buffer(place(13), 1, F), "rstd": buffer(place(14), 1, F),
        "residual_grad": None, "grad_weight": None, "grad_bias": None}, DF, "exceeds the grid range"),
    # recurrence
    (scan, {"gate": view(place(0), L([2, 5, 8]), B)}, IC, "recurrence gate must be float32"),
    (scan, {"state_in": view(place(3), L([2, 8]), B)}, IC, "recurrence state must be float32"),
    (scan, {"lengths": buffer(place(5), 2, np.int64)}, IC, "lengths must be uint32"),
    (scan, {"lengths": buffer(place(5), 3, U)}, LM, "2"),
    (scan, {"gate": view(place(0), L([2, 6, 8]), F)}, DF, "recurrence gate has shape"),
    (scan, {"state_out": view(place(4), L([2, 9]), F)}, DF, "recurrence state output has shape"),
    (scan, {"x": view(place(1), L([2, 40]), F)}, DF, "rank-3"),
    (scan, {"output": view(place(2), N([2, 5, 8], [0, 8, 1]), F)}, DF, "reach an element twice"),
    (scan, {"output": view(place(1), L([2, 5, 8]), F)}, DF, "must not overlap recurrence input"),
    (scan, {"output": view(place(0), L([2, 5, 8]), F)}, DF, "must not overlap recurrence gate"),
    (scan, {"state_out": view(place(3) + 4, L([2, 8]), F)}, DF, "must be the view of recurrence state"),
    (scan, {"state_out": view(place(2) + 8, L([2, 8]), F)}, DF, "must not overlap"),
    (scan, {"gate": view(place(0), L([65536, 1, 8]), F), "x": view(place(1), L([65536, 1, 8]), F),
            "output": view(place(2), L([65536, 1, 8]), F), "state_in": None, "state_out": None, "lengths": None}, DF,
     "at most 65535 sequences"),
    # recurrence, backward
    (scan_grad, {"h": view(place(2), L([2, 5, 8]), B)}, IC, "recurrence output must be float32"),
    (scan_grad, {"grad_state_in": view(place(8), L([2, 8]), B)}, IC, "gradient of the state must be float32"),
    (scan_grad, {"grad_out": view(place(3), L([2, 4, 8]), F)}, DF, "gradient of the recurrence output has shape"),
    (scan_grad, {"grad_gate": view(place(0), L([2, 5, 8]), F)}, DF, "must not overlap recurrence gate"),
    (scan_grad, {"grad_gate": view(place(5), L([2, 5, 8]), F)}, DF, "must not overlap"),
    (scan_grad, {"grad_x": view(place(3), L([2, 5, 8]), F)}, DF, "must not overlap gradient of the recurrence output"),
    (scan_grad, {"grad_state_in": view(place(7), L([2, 8]), F)}, DF, "must not overlap gradient of the state output"),
    # loss
    (loss, {"x": view(place(0), L([4, 8]), np.int8)}, IC, "float32 or bfloat16"),
    (loss, {"weight": view(place(1), L([9, 8]), B)}, IC, "vocabulary weight must be float32"),
    (loss, {"targets": buffer(place(2), 4, np.int64)}, IC, "targets must be uint32"),
    (loss, {"loss": buffer(place(3), 4, B)}, IC, "loss must be float32"),
    (loss, {"weight": view(place(1), L([9, 7]), F)}, DF, "vocabulary weight has shape"),
    (loss, {"targets": buffer(place(2), 5, U)}, LM, "4"),
    (loss, {"lse": buffer(place(4), 3, F)}, LM, "4"),
    (loss, {"lse": buffer(place(3), 4, F)}, DF, "must not overlap"),
    (loss, {"loss": buffer(place(0), 4, F)}, DF, "loss must not overlap loss input"),
    (loss, {"x": view(place(0), N([4, 8], [8, 0]), F)}, DF, "contiguous last dimension"),
    (loss, {"x": view(place(0), N([1 << 28, 8], [0, 1]), F, 8), "targets": buffer(place(2), 1 << 28, U),
            "loss": buffer(place(30), 1 << 28, F), "lse": None}, DF, "each is below 2^28"),
    (loss, {"x": view(place(0), L([4, (1 << 20) + 1]), F), "weight": view(place(1), L([9, (1 << 20) + 1]), F)}, DF,
     "at most 1048576"),
    # loss, backward
    (loss_grad, {"grad": buffer(place(4), 4, B)}, IC, "gradient of the loss must be float32"),
    (loss_grad, {"grad_x": view(place(5), L([4, 8]), B)}, IC, "gradient of the loss input must be float32"),
    (loss_grad, {"grad": buffer(place(4), 3, F)}, LM, "4"),
    (loss_grad, {"grad_weight": view(place(6), L([8, 9]), F)}, DF, "gradient of the vocabulary weight has shape"),
    (loss_grad, {"grad_x": view(place(0), L([4, 8]), F)}, DF, "must not overlap loss input"),
    (loss_grad, {"grad_weight": view(place(1), L([9, 8]), F)}, DF, "must not overlap vocabulary weight"),
    (loss_grad, {"grad_weight": view(place(5) + 16, L([9, 8]), F)}, DF, "must not overlap"),
]


@pytest.mark.parametrize("run,change,error,text", REFUSED, ids=[f"{r.method}-{i}" for i, (r, *_) in enumerate(REFUSED)])
def test_refused(run, change, error, text):
    with pytest.raises(error, match=None) as seen:
        run(**change)
    assert text in str(seen.value)


ALL = [norm, norm_grad, scan, scan_grad, loss, loss_grad]


@pytest.mark.parametrize("run", ALL, ids=[r.method for r in ALL])
def test_plans_refuse_the_same(run):
    """The prepare_* call has the same checks, and hands out no plan."""
    prepare = getattr(run.defaults["ops"], "prepare_" + run.method.removesuffix("_into"))
    for other, change, error, text in REFUSED:
        if other is run:
            with pytest.raises(error) as seen:
                prepare(NoDevice, **{k: v for k, v in {**run.defaults, **change}.items() if k != "ops"})
            assert text in str(seen.value)


@pytest.mark.parametrize("run", ALL, ids=[r.method for r in ALL])
def test_what_passes_the_checks_needs_a_device(run):
    """The operands that the refusals change are themselves fine."""
    with pytest.raises(hx.HephaestusError) as seen:
        run()
    assert "device" in str(seen.value)


def test_operands_left_out():
    """NULL layouts leave operands out; a buffer without a layout is no operand."""
    for run, names in ((norm, ("bias", "residual", "residual_out", "mean", "rstd")),
                       (norm_grad, ("residual_grad", "grad_weight", "grad_bias")),
                       (scan, ("state_in", "state_out", "lengths")),
                       (scan_grad, ("state_in", "grad_state_out", "grad_state_in", "lengths")), (loss, ("lse",)),
                       (loss_grad, ("grad_x", "grad_weight"))):
        with pytest.raises(hx.HephaestusError) as seen:
            run(**{name: None for name in names})
        assert "device" in str(seen.value)
    lib = hx.load_native()
    from hephaestus_amd import _ffi
    import ctypes
    lay = _ffi.layout_struct(L([4, 8]))
    lp = ctypes.byref(lay)
    status = lib.hx_linear_cross_entropy_backward(None, _ffi.lib() and 0, place(0), 32, lp, place(1), 32, lp, place(2), 4,
                                                  place(3), 4, place(4), 4, place(5), 32, None, None, 0, None, None)
    assert status != 0 and b"has a buffer and no layout" in lib.hx_last_error_message()


def test_in_place_as_documented():
    for run, change in ((norm, {"residual_out": norm.defaults["x"]}), (norm, {"residual_out": norm.defaults["residual"]}),
                        (norm_grad, {"grad_in": norm_grad.defaults["grad_out"]}),
                        (norm_grad, {"grad_in": norm_grad.defaults["residual_grad"]}),
                        (scan, {"state_out": scan.defaults["state_in"]})):
        with pytest.raises(hx.HephaestusError) as seen:
            run(**change)
        assert "device" in str(seen.value)


def test_views_between_each_other():
    """Gradients of gate and input side by side, as a projection's rows are."""
    pool = buffer(place(20), 2 * 5 * 16, F)
    halves = [StridedView(pool, N([2, 5, 8], [80, 16, 1], 8 * i)) for i in range(2)]
    with pytest.raises(hx.HephaestusError) as seen:
        scan_grad(grad_gate=halves[0], grad_x=halves[1])
    assert "device" in str(seen.value)
