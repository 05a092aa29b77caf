"""A small language model that mixes tokens by a gated recurrence, trained on the
device: an embedding, a layer norm, the recurrence and a head over the vocabulary.

    embedding of a token, 2·width -> layer norm -> gate | input, width each
        -> gated recurrence along the tokens (a state for each sequence)
        -> softmax cross entropy with the head's weights (logits are not kept)
    backward: the same operators' gradients in turn, each where the next one reads it

Every step of both passes is a plan that is prepared once for its buffers.  The
embedding's rows are gathered, and all parameters updated, on the host.

    python examples/recurrent_language_model.py [--steps 30]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import hephaestus_amd as hx  # noqa: E402
from hephaestus_amd import Layout, StridedView  # noqa: E402

EPSILON = 1e-5


class Model:
    """Parameters on the host in f32, in `dtype` on the device, and the plans of a
    training step for `batch` sequences of `tokens` tokens."""

    def __init__(self, device, vocab=256, width=64, batch=4, tokens=64, dtype=np.float32, seed=0):
        rng = np.random.default_rng(seed)
        self.device, self.dtype, self.vocab, self.shape = device, np.dtype(dtype), vocab, (batch, tokens, width)
        self.embedding = rng.normal(size=(vocab, 2 * width)).astype(np.float32)
        self.norm_weight = np.ones(2 * width, np.float32)
        # Gates that start open: the state remembers some ten tokens.
        self.norm_bias = np.repeat(np.array([2.0, 0.0], np.float32), width)
        self.head = (rng.normal(size=(vocab, width)) / np.sqrt(width)).astype(np.float32)
        self._prepare()

    def _prepare(self):
        device, (batch, tokens, width) = self.device, self.shape
        rows = batch * tokens

        def new(*shape):
            return StridedView(device.alloc_zeroed(self.dtype, int(np.prod(shape))), Layout.c_contiguous(shape))

        def floats(n):
            return device.alloc_zeroed(np.float32, n)

        def halves(view):  # gate | input of each token's row
            strides = (tokens * 2 * width, 2 * width, 1)
            return [StridedView(view.buffer, Layout.try_new((batch, tokens, width), strides, part * width))
                    for part in range(2)]

        def by_tokens(view):
            return StridedView(view.buffer, Layout.c_contiguous((batch, tokens, width)))

        self.x, y, self.dx, dy = (new(rows, 2 * width) for _ in range(4))
        h, dh = new(rows, width), new(rows, width)
        self.weight, self.bias = new(2 * width).buffer, new(2 * width).buffer
        self.head_view, self.dhead = new(self.vocab, width), new(self.vocab, width)
        mean, rstd, lse = floats(rows), floats(rows), floats(rows)
        self.loss, self.grad = floats(rows), floats(rows)
        self.dweight, self.dbias = floats(2 * width), floats(2 * width)
        self.targets = device.alloc_zeroed(np.uint32, rows)
        self.lengths = device.alloc_zeroed(np.uint32, batch)
        (gate, u), (dgate, du) = halves(y), halves(dy)
        norm, mix, loss = hx.RocmLayerNormOps(), hx.RocmRecurrenceOps(), hx.RocmLossOps()
        self.plans = [
            norm.prepare_layer_norm(device, self.x, self.weight, self.bias, EPSILON, y, mean=mean, rstd=rstd),
            mix.prepare_gated_recurrence(device, gate, u, by_tokens(h), lengths=self.lengths),
            loss.prepare_linear_cross_entropy(device, h, self.head_view, self.targets, self.loss, lse),
            loss.prepare_linear_cross_entropy_backward(device, h, self.head_view, self.targets, lse, self.grad,
                                                       grad_x=dh, grad_weight=self.dhead),
            mix.prepare_gated_recurrence_backward(device, gate, u, by_tokens(h), by_tokens(dh), dgate, du,
                                                  lengths=self.lengths),
            norm.prepare_layer_norm_backward(device, dy, self.x, self.weight, mean, rstd, self.dx,
                                             grad_weight=self.dweight, grad_bias=self.dbias),
        ]

    def _put(self, buffer, values):
        values = np.ascontiguousarray(values, np.float32).reshape(-1)
        self.device.write_buffer(buffer, hx.bfloat16_from_float32(values) if self.dtype == hx.bfloat16 else values)

    def _get(self, buffer, shape):
        host = self.device.download_owned(buffer)
        return (hx.float32_from_bfloat16(host) if host.dtype == hx.bfloat16 else host).reshape(shape)

    def step(self, text, lengths):
        """(mean loss, gradients by parameter) of [batch, tokens + 1] words, of which
        a sequence has `lengths` words to predict."""
        batch, tokens, width = self.shape
        words, following = text[:, :-1], text[:, 1:]
        is_there = np.arange(tokens)[None] < np.asarray(lengths)[:, None]
        self._put(self.x.buffer, self.embedding[words])
        self._put(self.weight, self.norm_weight)
        self._put(self.bias, self.norm_bias)
        self._put(self.head_view.buffer, self.head)
        self.device.write_buffer(self.targets, np.where(is_there, following, hx.NO_TARGET).astype(np.uint32).reshape(-1))
        self.device.write_buffer(self.lengths, np.asarray(lengths, np.uint32))
        self.device.write_buffer(self.grad, (is_there / max(1, is_there.sum())).astype(np.float32).reshape(-1))
        hx.submit_prepared_reduction_batch(self.plans)
        self.device.synchronize()
        dx = self._get(self.dx.buffer, (batch * tokens, 2 * width))
        embedding = np.zeros_like(self.embedding)
        np.add.at(embedding, words.reshape(-1), dx)
        losses = self.device.download_owned(self.loss).astype(np.float64)
        return losses.sum() / max(1, is_there.sum()), {
            "embedding": embedding, "norm_weight": self.device.download_owned(self.dweight),
            "norm_bias": self.device.download_owned(self.dbias), "head": self._get(self.dhead.buffer, self.head.shape)}

    def update(self, gradients, rate):
        for name, gradient in gradients.items():
            setattr(self, name, getattr(self, name) - np.float32(rate) * gradient)


def text_of(batch, tokens, vocab, seed=0):
    """Words that follow from the one before, but for one in eight."""
    rng = np.random.default_rng(seed)
    follows = np.random.default_rng(0).permutation(vocab)  # the same in every text
    text = np.empty((batch, tokens + 1), np.int64)
    text[:, 0] = rng.integers(0, vocab, batch)
    for t in range(tokens):
        text[:, t + 1] = np.where(rng.random(batch) < 1 / 8, rng.integers(0, vocab, batch), follows[text[:, t]])
    return text, rng.integers(tokens // 2, tokens + 1, batch)


def main():
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=30)
    args = parser.parse_args()
    device = hx.RocmDevice.try_default()
    model = Model(device, dtype=hx.bfloat16)
    for step in range(args.steps):
        loss, gradients = model.step(*text_of(4, 64, model.vocab, seed=step))
        model.update(gradients, rate=8.0)
        print(f"step {step}: loss {loss:.3f}", flush=True)


if __name__ == "__main__":
    main()
