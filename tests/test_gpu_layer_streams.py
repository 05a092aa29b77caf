"""The layer operators on callers' streams, under stream capture, and as plans
that re-read their operands."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
import test_gpu_linear_attention as attention
import test_gpu_matmul_i8 as matmul
import test_gpu_norm_quantize as norm
from layer_reference import padded, rounded, vector
from test_gpu_capture import Capture, Stream

pytestmark = pytest.mark.gpu


class Layer:
    """One plan of each operator over buffers that a test rewrites: small and
    large products, single tokens and a split prompt."""

    def __init__(self, device):
        self.device, t = device, hx.bfloat16
        self.cases = []
        x, r, w = (rounded(np.zeros(s), t) for s in ((33, 1000), (33, 1000), 1000))
        vx, vr = padded(device, x)[0], padded(device, r)[0]
        vq, read_q = padded(device, np.zeros(x.shape, np.int8))
        vh, read_h = padded(device, x)
        vw, vs = vector(device, w), device.alloc_zeroed(np.float32, 33)
        args = (device, vx, vw, 1e-5, vq, vs, vr, vh)

        def inputs(rng):
            return tuple(rounded(rng.normal(size=a.shape), t) for a in (x, r, w))

        def verify(ins):
            norm.check(*ins, (read_h(), read_q(), device.download_owned(vs)))

        ops = hx.RocmNormOps()
        self.add((vx.buffer, vr.buffer, vw), inputs, ops.prepare_rms_norm_quantize(*args),
                 lambda s, args=args: ops.rms_norm_quantize_into(*args, stream=s), verify)
        for m, n, k in ((3, 700, 2048), (300, 520, 384)):
            self.add_matmul(m, n, k)
        for tokens in (1, 300):
            self.add_attention(tokens)

    def add(self, buffers, inputs, plan, call, verify):
        self.cases.append((buffers, inputs, plan, call, verify))

    def add_matmul(self, m, n, k):
        device, zero = self.device, matmul.operands(m, n, k)
        va, vb = padded(device, zero[0])[0], padded(device, zero[1])[0]
        sa, sb = vector(device, zero[2]), vector(device, zero[3])
        vo, read = padded(device, np.zeros((m, n), np.float32))
        args, ops = (device, va, sa, vb, sb, vo), hx.RocmMatrixOps()
        self.add((va.buffer, vb.buffer, sa, sb), lambda rng: matmul.operands(m, n, k, int(rng.integers(1 << 20))),
                 ops.prepare_matmul_i8(*args), lambda s: ops.matmul_i8_into(*args, stream=s),
                 lambda ins: matmul.check(*ins, read()))

    def add_attention(self, tokens):
        device, t = self.device, hx.bfloat16
        zero = attention.operands(t, 1, tokens, 2, 1, 64, 48)
        views = [padded(device, x)[0] for x in zero[:3]]
        decay, first = vector(device, zero[3]), padded(device, zero[4])[0]
        vo, read_o = padded(device, rounded(np.zeros((1, tokens, 2, 48)), t))
        vs, read_s = padded(device, np.zeros_like(zero[4]))
        args, ops = (device, *views, decay, vo, None, first, vs), hx.RocmLinearAttentionOps()
        self.add((*(v.buffer for v in views), decay, first.buffer),
                 lambda rng: attention.operands(t, 1, tokens, 2, 1, 64, 48, int(rng.integers(1 << 20))),
                 ops.prepare_linear_attention(*args), lambda s: ops.linear_attention_into(*args, stream=s),
                 lambda ins: attention.check(*ins, None, (read_o(), read_s())))

    def write(self, seed):
        rng, ins = np.random.default_rng(seed), []
        for buffers, inputs, *_ in self.cases:
            ins.append(inputs(rng))
            for b, x in zip(buffers, ins[-1]):
                self.device.write_buffer(b, np.ascontiguousarray(x).reshape(-1))
        return ins

    def verify(self, ins):
        for (*_, verify), x in zip(self.cases, ins):
            verify(x)


@pytest.fixture(scope="module")
def layer(device):
    return Layer(device)


def test_plans_read_their_operands_anew(device, layer):
    for seed in (1, 2):
        ins = layer.write(seed)
        for _, _, plan, _, _ in layer.cases:
            plan.dispatch()
        device.synchronize()
        layer.verify(ins)


def test_immediate_calls_on_a_callers_stream(device, layer):
    stream = Stream()
    try:
        for seed in (3, 4):
            ins = layer.write(seed)
            for _, _, _, call, _ in layer.cases:
                call(stream.value)
            stream.sync()
            layer.verify(ins)
    finally:
        stream.close(device)


def test_plans_under_capture(device, layer):
    """A graph of all plans, replayed with new inputs, eager calls between."""
    stream = Stream()
    capture = Capture(stream)
    try:
        with capture:
            for _, _, plan, _, _ in layer.cases:
                plan.dispatch(stream.value)
        for seed in (5, 6, 7, 8):
            ins = layer.write(seed)
            capture.replay()
            layer.verify(ins)
            ins = layer.write(seed + 100)
            for _, _, plan, call, _ in layer.cases:
                plan.dispatch()
            device.synchronize()
            layer.verify(ins)
    finally:
        capture.destroy()
        stream.close(device)


def test_immediate_calls_that_take_scratch_refuse_capture(device, layer):
    stream = Stream()
    capture = Capture(stream)
    try:
        with capture:
            for _, _, plan, call, _ in layer.cases[1:]:
                with pytest.raises(hx.DispatchFailed):
                    call(stream.value)
            layer.cases[0][2].dispatch(stream.value)
        ins = layer.write(9)
        capture.replay()
        layer.cases[0][4](ins[0])
    finally:
        capture.destroy()
        stream.close(device)


def test_other_owners_memory(device):
    """A borrowed buffer is read and written in place, and never freed."""
    own = device.upload(np.arange(256, dtype=np.float32))
    lent = device.borrow(own.ptr, np.float32, 256, owner=own)
    view = hx.StridedView(lent, hx.Layout.c_contiguous([2, 128]))
    q, s = device.alloc_zeroed(np.int8, 256), device.alloc_zeroed(np.float32, 2)
    hx.RocmNormOps().rms_norm_quantize_into(device, view, device.upload(np.ones(128, np.float32)), 0.0,
                                            hx.StridedView(q, hx.Layout.c_contiguous([2, 128])), s)
    device.synchronize()
    del lent, view
    assert np.array_equal(device.download_owned(own), np.arange(256, dtype=np.float32))
    assert device.download_owned(q)[255] == 127
