"""The example layer: a prompt followed by single tokens gives what all tokens
at once give, and both give what the layer's formula gives in 64 bits."""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import pytest

import hephaestus_amd as hx
from layer_reference import as_float64, linear_attention, norm_quantize

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
import linear_attention_layer as example  # noqa: E402

pytestmark = pytest.mark.gpu

SIZES = {"batch": 2, "width": 192, "heads": 4, "head": 32}


def reference(layer, x, residual):
    """The layer in 64 bits, with its roundings to 8 bits and to bf16."""
    batch, tokens, width = x.shape
    inner = layer.heads * layer.head

    def bf16(values):
        return as_float64(hx.bfloat16_from_float32(values.astype(np.float32)))

    def product(values, weight, matrix, extra=None):
        _, steps, s = norm_quantize(hx.bfloat16_from_float32(values.astype(np.float32)),
                                    extra, weight, layer.epsilon)
        return bf16(s[:, None] * (np.rint(steps) @ matrix.values.T.astype(np.float64)) * matrix.scales)

    qkv = product(x.reshape(-1, width), layer.norm_in, layer.to_qkv,
                  hx.bfloat16_from_float32(residual.reshape(-1, width)))
    q, k, v = (qkv[:, i * inner:(i + 1) * inner].reshape(batch, tokens, layer.heads, layer.head).astype(np.float32)
               for i in range(3))
    o = linear_attention(q, k, v, layer.log_decay, layer.head ** -0.5)[0]
    return product(bf16(o).reshape(-1, inner), layer.norm_out, layer.to_out).reshape(x.shape)


def test_prompt_then_tokens(device):
    served, whole = example.serve(device, tokens=70, steps=5, **SIZES)
    layer = example.Layer(device, **SIZES)
    rng = np.random.default_rng(1)
    x, residual = rng.normal(size=(2, 2, 75, 192)).astype(np.float32)
    want = reference(layer, x, residual)
    # Roundings to bf16 move the attention's outputs by up to 2^-8 each, and those
    # by a step of 1/127 at most that fall on the other side of a half: together
    # within two hundredths in the norm.
    for got in (served, whole):
        assert np.linalg.norm(got - want) <= 0.02 * np.linalg.norm(want)
    assert np.linalg.norm(served - whole) <= 0.02 * np.linalg.norm(whole)
