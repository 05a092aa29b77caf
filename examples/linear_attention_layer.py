"""One layer of a linear-attention model, served in 8 bits: a prompt of several
sequences, then one token at a time from the state that the prompt left.

    x, residual -> RMS norm, 8 bits -> product -> q | k | v
                -> linear attention with a decay for each head (state kept)
                -> RMS norm, 8 bits -> product -> y     (x of the next layer)

Every step is a plan that is prepared once for its buffers and dispatched for
each call; the attention reads q, k and v where the product wrote them.

    python examples/linear_attention_layer.py [--tokens 512] [--steps 16]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import hephaestus_amd as hx  # noqa: E402
from hephaestus_amd import Layout, StridedView  # noqa: E402


class Weights:
    """8-bit weights with a scale for each channel, on the device."""

    def __init__(self, device, matrix):
        scales = np.abs(matrix).max(axis=1) / 127
        self.values = np.rint(matrix / scales[:, None]).astype(np.int8)
        self.scales = scales.astype(np.float32)
        self.view = StridedView(device.upload(self.values), Layout.c_contiguous(matrix.shape))
        self.scale_buffer = device.upload(self.scales)


class Layer:
    """The weights of a layer and its state for `batch` sequences."""

    def __init__(self, device, batch=4, width=512, heads=8, head=64, epsilon=1e-5, seed=0):
        rng = np.random.default_rng(seed)
        self.device, self.batch, self.width, self.heads, self.head = device, batch, width, heads, head
        self.epsilon = epsilon
        inner = heads * head
        self.norm_in = hx.bfloat16_from_float32(rng.uniform(0.5, 1.5, width))
        self.norm_out = hx.bfloat16_from_float32(rng.uniform(0.5, 1.5, inner))
        self.to_qkv = Weights(device, rng.normal(size=(3 * inner, width)) / np.sqrt(width))
        self.to_out = Weights(device, rng.normal(size=(width, inner)) / np.sqrt(inner))
        # Heads that remember from 4 to 512 tokens.
        self.log_decay = np.log1p(-np.exp2(-np.linspace(2, 9, heads))).astype(np.float32)
        self.norm_in_buffer, self.norm_out_buffer = device.upload(self.norm_in), device.upload(self.norm_out)
        self.decay_buffer = device.upload(self.log_decay)
        shape = (batch, heads, head, head)
        self.state = StridedView(device.alloc_zeroed(np.float32, int(np.prod(shape))), Layout.c_contiguous(shape))

    def forward(self, tokens):
        """The layer for `tokens` tokens of each sequence."""
        return Forward(self, tokens)


class Forward:
    """A layer's plans and buffers for one number of tokens."""

    def __init__(self, layer, tokens):
        device, inner = layer.device, layer.heads * layer.head
        rows = layer.batch * tokens
        self.device, self.shape = device, (layer.batch, tokens, layer.width)

        def new(dtype, *shape):
            return StridedView(device.alloc_zeroed(dtype, int(np.prod(shape))), Layout.c_contiguous(shape))

        self.x, self.residual = new(hx.bfloat16, rows, layer.width), new(hx.bfloat16, rows, layer.width)
        self.h, self.y = new(hx.bfloat16, rows, layer.width), new(hx.bfloat16, rows, layer.width)
        qkv, o = new(hx.bfloat16, rows, 3 * inner), new(hx.bfloat16, rows, inner)
        quantized = [new(np.int8, rows, n) for n in (layer.width, inner)]
        scales = [device.alloc_zeroed(np.float32, rows) for _ in range(2)]

        # q, k and v inside the product's rows: [batch, tokens, heads, head].
        shape = (layer.batch, tokens, layer.heads, layer.head)
        strides = (tokens * 3 * inner, 3 * inner, layer.head, 1)
        q, k, v = (StridedView(qkv.buffer, Layout.try_new(shape, strides, part * inner)) for part in range(3))
        out = StridedView(o.buffer, Layout.c_contiguous(shape))
        norm, matrix, attention = hx.RocmNormOps(), hx.RocmMatrixOps(), hx.RocmLinearAttentionOps()
        self.plans = [
            norm.prepare_rms_norm_quantize(device, self.x, layer.norm_in_buffer, layer.epsilon, quantized[0], scales[0],
                                           residual=self.residual, residual_out=self.h),
            matrix.prepare_matmul_i8(device, quantized[0], scales[0], layer.to_qkv.view, layer.to_qkv.scale_buffer, qkv),
            attention.prepare_linear_attention(device, q, k, v, layer.decay_buffer, out, state_in=layer.state,
                                               state_out=layer.state),
            norm.prepare_rms_norm_quantize(device, o, layer.norm_out_buffer, layer.epsilon, quantized[1], scales[1]),
            matrix.prepare_matmul_i8(device, quantized[1], scales[1], layer.to_out.view, layer.to_out.scale_buffer,
                                     self.y),
        ]

    def __call__(self, x, residual):
        """(y, residual) of [batch, tokens, width] arrays in f32."""
        for view, host in ((self.x, x), (self.residual, residual)):
            self.device.write_buffer(view.buffer, hx.bfloat16_from_float32(host).reshape(-1))
        hx.submit_prepared_reduction_batch(self.plans)
        self.device.synchronize()
        return tuple(hx.float32_from_bfloat16(self.device.download_owned(v.buffer)).reshape(self.shape)
                     for v in (self.y, self.h))


def serve(device, tokens=512, steps=16, **sizes):
    """A prompt and then single tokens, and the same tokens all at once: the two
    outputs, [batch, tokens + steps, width]."""
    layer = Layer(device, **sizes)
    rng = np.random.default_rng(1)
    x, residual = rng.normal(size=(2, layer.batch, tokens + steps, layer.width)).astype(np.float32)
    parts = [layer.forward(tokens)(x[:, :tokens], residual[:, :tokens])[0]]
    step = layer.forward(1)
    for t in range(tokens, tokens + steps):
        parts.append(step(x[:, t:t + 1], residual[:, t:t + 1])[0])
    fresh = Layer(device, **sizes)  # the same weights, an empty state
    return np.concatenate(parts, axis=1), fresh.forward(tokens + steps)(x, residual)[0]


def main():
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--tokens", type=int, default=512)
    parser.add_argument("--steps", type=int, default=16)
    args = parser.parse_args()
    device = hx.RocmDevice.try_default()
    served, whole = serve(device, args.tokens, args.steps)
    off = np.linalg.norm(served - whole) / np.linalg.norm(whole)
    print(f"{served.shape[0]} sequences of {args.tokens} tokens and {args.steps} steps: "
          f"outputs {served.shape}, {off:.2e} from the same tokens at once")


if __name__ == "__main__":
    main()
