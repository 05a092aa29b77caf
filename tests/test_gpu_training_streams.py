"""The training operators as plans that re-read their operands, on callers'
streams, under stream capture, and as a run of them together: a layer norm, a
recurrence, a residual and a loss, forward and backward."""
from __future__ import annotations

import threading

import numpy as np
import pytest

import hephaestus_amd as hx
import test_gpu_cross_entropy as entropy
import test_gpu_gated_recurrence as recurrence
from layer_reference import padded, rounded, vector
from test_gpu_capture import Capture, Stream
from test_gpu_layer_norm import operands as norm_operands, stats_of
from training_reference import (cross_entropy, cross_entropy_backward, gated_recurrence, gated_recurrence_backward,
                                layer_norm, layer_norm_backward, near)

pytestmark = pytest.mark.gpu


class Operators:
    """One plan of each operator and direction over buffers that a test rewrites: a
    recurrence of few and one of many tokens, a small and a larger loss."""

    def __init__(self, device):
        self.device, self.cases = device, []
        for t in (hx.bfloat16, np.float32):
            self.add_norm(t, 300, 520)
            self.add_recurrence(t, 2, 1, 70)
            self.add_recurrence(t, 1, 700, 130)
            self.add_loss(t, 7, 300, 64)
            self.add_loss(t, 200, 400, 72)

    def add(self, ops, method, views, outputs, inputs, verify, scratch):
        """`views` and `outputs` by argument name; inputs(rng) gives the arrays of `views`."""
        args = {**views, **{k: v for k, (v, _) in outputs.items()}}
        self.cases.append({
            "views": views, "inputs": inputs, "verify": verify, "scratch": scratch, "method": method,
            "outputs": outputs, "plan": getattr(ops, f"prepare_{method}")(self.device, **args),
            "call": lambda stream: getattr(ops, f"{method}_into")(self.device, **args, stream=stream)})

    def out(self, t, *shape):
        return padded(self.device, rounded(np.zeros(shape), t))

    def vec(self, n):
        b = vector(self.device, np.zeros(n, np.float32))
        return b, lambda: self.device.download_owned(b)

    def view(self, a):
        return padded(self.device, a)[0]

    def add_norm(self, t, rows, cols):
        x, r, w, b, dy, past = norm_operands(t, rows, cols)
        ops = hx.RocmLayerNormOps()
        views = {"x": self.view(x), "weight": vector(self.device, w), "bias": vector(self.device, b), "residual": self.view(r)}
        outputs = {"output": self.out(t, rows, cols), "residual_out": self.out(t, rows, cols), "mean": self.vec(rows),
                   "rstd": self.vec(rows)}

        def inputs(seed):
            a = norm_operands(t, rows, cols, seed)
            return {"x": a[0], "weight": a[2], "bias": a[3], "residual": a[1]}

        def verify(a, got):
            value, bound = layer_norm(a["x"], a["residual"], a["weight"], a["bias"], 1e-5)
            for name, of in (("output", "y"), ("residual_out", "h"), ("mean", "mean"), ("rstd", "rstd")):
                near(got[name], value[of], bound[of], of)

        class Ops:  # epsilon bound
            @staticmethod
            def layer_norm_into(device, stream=None, **k):
                ops.layer_norm_into(device, epsilon=1e-5, stream=stream, **k)

            @staticmethod
            def prepare_layer_norm(device, **k):
                return ops.prepare_layer_norm(device, epsilon=1e-5, **k)

        self.add(Ops, "layer_norm", views, outputs, inputs, verify, False)
        mean, rstd = stats_of(x)
        views = {"grad_out": self.view(dy), "x": self.view(x), "weight": vector(self.device, w),
                 "mean": vector(self.device, mean), "rstd": vector(self.device, rstd), "residual_grad": self.view(past)}
        outputs = {"grad_in": self.out(t, rows, cols), "grad_weight": self.vec(cols), "grad_bias": self.vec(cols)}

        def inputs_back(seed):
            a = norm_operands(t, rows, cols, seed)
            mean, rstd = stats_of(a[0])
            return {"grad_out": a[4], "x": a[0], "weight": a[2], "mean": mean, "rstd": rstd, "residual_grad": a[5]}

        def verify_back(a, got):
            value, bound = layer_norm_backward(a["grad_out"], a["x"], a["weight"], a["mean"], a["rstd"], a["residual_grad"])
            for name, of in (("grad_in", "dh"), ("grad_weight", "dw"), ("grad_bias", "db")):
                near(got[name], value[of], bound[of], of)

        self.add(ops, "layer_norm_backward", views, outputs, inputs_back, verify_back, True)

    def add_recurrence(self, t, batch, tokens, channels):
        shape, ops = (batch, tokens, channels), hx.RocmRecurrenceOps()

        def inputs(seed):
            gate, x, _, first, _ = recurrence.operands(t, *shape, seed)
            return {"gate": gate, "x": x, "state_in": first}

        def verify(a, got):
            value, bound = gated_recurrence(a["gate"], a["x"], a["state_in"])
            near(got["output"], value["h"], bound["h"], "h")
            near(got["state_out"], value["last"], bound["last"], "last")

        a = inputs(0)
        self.add(ops, "gated_recurrence", {k: self.view(v) for k, v in a.items()},
                 {"output": self.out(t, *shape), "state_out": self.out(np.float32, batch, channels)}, inputs, verify,
                 tokens > 32)

        def inputs_back(seed):
            gate, x, dy, first, dlast = recurrence.operands(t, *shape, seed)
            h = rounded(gated_recurrence(gate, x, first)[0]["h"], t)
            return {"gate": gate, "x": x, "h": h, "grad_out": dy, "state_in": first, "grad_state_out": dlast}

        def verify_back(a, got):
            value, bound = gated_recurrence_backward(a["gate"], a["x"], a["h"], a["grad_out"], a["state_in"],
                                                     a["grad_state_out"])
            for name, of in (("grad_gate", "dgate"), ("grad_x", "dx"), ("grad_state_in", "dfirst")):
                near(got[name], value[of], bound[of], of)

        a = inputs_back(0)
        self.add(ops, "gated_recurrence_backward", {k: self.view(v) for k, v in a.items()},
                 {"grad_gate": self.out(t, *shape), "grad_x": self.out(t, *shape),
                  "grad_state_in": self.out(np.float32, batch, channels)}, inputs_back, verify_back, tokens > 32)

    def add_loss(self, t, rows, vocab, width):
        ops = hx.RocmLossOps()

        def place(a):
            return {k: self.view(v) if v.ndim == 2 else vector(self.device, v) for k, v in a.items()}

        def inputs(seed):
            x, w, targets, _ = entropy.operands(t, rows, vocab, width, seed)
            return {"x": x, "weight": w, "targets": targets}

        def verify(a, got):
            value, bound = cross_entropy(a["x"], a["weight"], a["targets"])
            for name in got:
                near(got[name], value[name], bound[name], name)

        self.add(ops, "linear_cross_entropy", place(inputs(0)), {"loss": self.vec(rows), "lse": self.vec(rows)}, inputs,
                 verify, True)

        def inputs_back(seed):
            x, w, targets, grad = entropy.operands(t, rows, vocab, width, seed)
            return {"x": x, "weight": w, "targets": targets, "lse": entropy.lse_of(x, w), "grad": grad}

        def verify_back(a, got):
            value, bound = cross_entropy_backward(*a.values())
            near(got["grad_x"], value["dx"], bound["dx"], "dx")
            near(got["grad_weight"], value["dw"], bound["dw"], "dw")

        self.add(ops, "linear_cross_entropy_backward", place(inputs_back(0)),
                 {"grad_x": self.out(t, rows, width), "grad_weight": self.out(t, vocab, width)}, inputs_back, verify_back,
                 True)

    def write(self, seed):
        ins = []
        for case in self.cases:
            ins.append(case["inputs"](seed))
            for name, array in ins[-1].items():
                v = case["views"][name]
                self.device.write_buffer(getattr(v, "buffer", v), np.ascontiguousarray(array).reshape(-1))
            for _, (v, _) in case["outputs"].items():
                b = getattr(v, "buffer", v)
                self.device.write_buffer(b, np.zeros(len(b), b.dtype))
        return ins

    def verify(self, ins):
        for case, a in zip(self.cases, ins):
            case["verify"](a, {name: read() for name, (_, read) in case["outputs"].items()})


@pytest.fixture(scope="module")
def operators(device):
    return Operators(device)


def test_plans_read_their_operands_anew(device, operators):
    for seed in (1, 2):
        ins = operators.write(seed)
        for case in operators.cases:
            case["plan"].dispatch()
        device.synchronize()
        operators.verify(ins)


def test_immediate_calls_on_a_callers_stream(device, operators):
    stream = Stream()
    try:
        for seed in (3, 4):
            ins = operators.write(seed)
            for case in operators.cases:
                case["call"](stream.value)
            stream.sync()
            operators.verify(ins)
    finally:
        stream.close(device)


def test_two_streams_at_once(device, operators):
    """Immediate calls of two threads, a stream each: their scratch is their own.
    The cases are split between them, as they write to their own buffers."""
    streams = [Stream(), Stream()]
    try:
        ins = operators.write(11)

        def run(i):
            for _ in range(3):
                for case in operators.cases[i::2]:
                    case["call"](streams[i].value)

        threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for s in streams:
            s.sync()
        operators.verify(ins)
    finally:
        for s in streams:
            s.close(device)


def test_plans_under_capture(device, operators):
    """A graph of all plans, replayed with new inputs, eager calls between."""
    stream = Stream()
    capture = Capture(stream)
    try:
        with capture:
            for case in operators.cases:
                case["plan"].dispatch(stream.value)
        for seed in (5, 6, 7, 8):
            ins = operators.write(seed)
            capture.replay()
            operators.verify(ins)
            ins = operators.write(seed + 100)
            for case in operators.cases:
                case["plan"].dispatch()
            device.synchronize()
            operators.verify(ins)
    finally:
        capture.destroy()
        stream.close(device)


def test_immediate_calls_under_capture(device, operators):
    """Those that take scratch refuse; the others are captured."""
    stream = Stream()
    capture = Capture(stream)
    try:
        with capture:
            for case in operators.cases:
                if case["scratch"]:
                    with pytest.raises(hx.DispatchFailed):
                        case["call"](stream.value)
                else:
                    case["call"](stream.value)
        ins = operators.write(9)
        capture.replay()
        for case, a in zip(operators.cases, ins):
            if not case["scratch"]:
                case["verify"](a, {name: read() for name, (_, read) in case["outputs"].items()})
    finally:
        capture.destroy()
        stream.close(device)
