"""Which views of one buffer the layer operators take together: those that share
no element, however they lie within one another.  Checks run before a device is
touched, so these need none."""
from __future__ import annotations

import itertools

import numpy as np
import pytest

import hephaestus_amd as hx
from hephaestus_amd import Layout, StridedView
from test_layer_refusals import B, F, attention, buffer, matmul, norm, view

N = Layout.try_new


def refusal(call, **change):
    """The message of a refused call; None where it got as far as the missing device."""
    with pytest.raises(hx.HephaestusError) as e:
        call(**change)
    return None if "device" in str(e.value) else str(e.value)


def elements(layout):
    """The elements that a view reaches, as a list with one entry an index."""
    return [layout.offset + sum(i * s for i, s in zip(index, layout.strides))
            for index in itertools.product(*map(range, layout.shape))]


def random_layout(rng, rank, length):
    """A view within `length` elements whose last dimension is contiguous."""
    while True:
        shape = [int(n) for n in rng.integers(1, 5, rank)]
        strides = [*(int(s) for s in rng.choice([-40, -24, -12, -8, -5, 0, 3, 4, 6, 8, 12, 16, 24, 30, 48, 60], rank - 1)), 1]
        offset = int(rng.integers(0, length))
        low = offset + sum(min(0, s * (n - 1)) for s, n in zip(strides, shape))
        high = offset + sum(max(0, s * (n - 1)) for s, n in zip(strides, shape))
        if 0 <= low and high < length:
            return N(shape, strides, offset)


def test_random_views_of_one_buffer():
    """Against the elements, one by one."""
    rng, taken, refused = np.random.default_rng(1), 0, 0
    for _ in range(4000):
        x = random_layout(rng, 2, 200)
        out = random_layout(rng, 2, 200)
        out = N(x.shape, out.strides, out.offset) if rng.random() < 0.7 else N(x.shape, x.strides, out.offset)
        reached = elements(out)
        if not 0 <= min(reached) <= max(reached) < 200 or len(set(reached)) < len(reached):
            continue
        rows, cols = x.shape
        said = refusal(norm, x=view(0x1000000, x, F, 200), residual_out=view(0x1000000, out, F, 200), residual=None,
                       weight=buffer(0x2000000, cols, F), scales=buffer(0x4000000, rows, F),
                       quantized=view(0x3000000, Layout.c_contiguous([rows, cols]), np.int8))
        shared = bool(set(elements(x)) & set(reached)) and elements(x) != reached
        assert (said is not None) == shared, (x, out, said)
        taken, refused = taken + (not shared), refused + shared
    assert taken > 300 and refused > 300


def test_random_states_of_one_pool():
    """Four dimensions, at every order of their strides."""
    rng, taken, refused = np.random.default_rng(2), 0, 0
    for _ in range(4000):
        first = random_layout(rng, 4, 300)
        last = random_layout(rng, 4, 300)
        last = N(first.shape, last.strides if rng.random() < 0.3 else first.strides, last.offset)
        reached = elements(last)
        if not 0 <= min(reached) <= max(reached) < 300 or len(set(reached)) < len(reached):
            continue
        b, h, dk, dv = first.shape
        said = refusal(attention, q=view(0x1000000, Layout.c_contiguous([b, 1, h, dk]), F),
                       k=view(0x2000000, Layout.c_contiguous([b, 1, h, dk]), F),
                       v=view(0x3000000, Layout.c_contiguous([b, 1, h, dv]), F),
                       output=view(0x5000000, Layout.c_contiguous([b, 1, h, dv]), F),
                       log_decay=buffer(0x4000000, h, F), lengths=None,
                       state_in=view(0x6000000, first, F, 300), state_out=view(0x6000000, last, F, 300))
        shared = bool(set(elements(first)) & set(reached)) and elements(first) != reached
        assert (said is not None) == shared, (first, last, said)
        taken, refused = taken + (said is None), refused + shared
    assert taken > 200 and refused > 200


def packed(at, width, tokens=5, heads=4, row=256, batch=2):
    return N([batch, tokens, heads, width], [tokens * row, row, width, 1], at)


@pytest.mark.parametrize("dtype", [F, B])
def test_an_output_beside_its_operands_in_one_row(dtype):
    """q | k | v | o of each token: 4 heads of 8 and 16 wide in rows of 256."""
    def part(at, width):
        return view(0x1000000, packed(at, width), dtype, 2 * 5 * 256)

    ops = {"q": part(0, 8), "k": part(32, 8), "v": part(64, 16)}
    assert refusal(attention, **ops, output=part(128, 16)) is None
    assert refusal(attention, **ops, output=part(192, 16)) is None
    assert "must not overlap the value" in refusal(attention, **ops, output=part(127, 16))
    before = view(0x1000000, packed(64, 8), dtype, 2 * 5 * 256)
    assert "must not overlap the query" in refusal(attention, **{**ops, "q": before}, output=part(95, 16))


def test_state_slots_of_one_pool():
    """Two slots a sequence, one read and one written, and the same one in place."""
    def slot(i, heads=4):
        return view(0x6000000, N([2, heads, 8, 16], [2 * heads * 128, 128, 16, 1], i * heads * 128), F, 4 * heads * 128)

    assert refusal(attention, state_in=slot(0), state_out=slot(1)) is None
    assert refusal(attention, state_in=slot(1), state_out=slot(0)) is None
    assert refusal(attention, state_in=slot(1), state_out=slot(1)) is None
    shifted = view(0x6000000, N([2, 4, 8, 16], [1024, 128, 16, 1], 512 - 16), F, 2048)
    assert "view of the state" in refusal(attention, state_in=slot(0), state_out=shifted)


def test_bytes_between_wider_elements():
    """8-bit rows and their f32 or bf16 neighbours in one allocation."""
    x = N([4, 64], [96, 1])  # f32 rows of 384 bytes, the last 128 of them free
    free = view(0x1000000, N([4, 64], [384, 1], 256), np.int8, 4 * 384)
    assert refusal(norm, x=view(0x1000000, x, F, 384), quantized=free) is None
    into = view(0x1000000, N([4, 64], [384, 1], 255), np.int8, 4 * 384)
    assert "must not overlap the norm input" in refusal(norm, x=view(0x1000000, x, F, 384), quantized=into)
    out = N([4, 6], [32, 1], 16)  # f32, after the 64 bytes of a's rows
    assert refusal(matmul, a=view(0x1000000, N([4, 64], [128, 1]), np.int8, 512), output=view(0x1000000, out, F, 128)) is None
    assert "must not overlap matmul a" in refusal(
        matmul, a=view(0x1000000, N([4, 65], [128, 1]), np.int8, 512), b=view(0x3000000, Layout.c_contiguous([6, 65]), np.int8),
        output=view(0x1000000, out, F, 128))


def test_outputs_whose_strides_cross():
    """Against the elements, one by one: a view is an output if it reaches none twice."""
    rng, taken, refused, crossed = np.random.default_rng(3), 0, 0, 0
    for _ in range(6000):
        out = random_layout(rng, 4, 300)
        b, h, dk, dv = out.shape
        reached = elements(out)
        once = len(set(reached)) == len(reached)
        said = refusal(attention, q=view(0x1000000, Layout.c_contiguous([b, 1, h, dk]), F),
                       k=view(0x2000000, Layout.c_contiguous([b, 1, h, dk]), F),
                       v=view(0x3000000, Layout.c_contiguous([b, 1, h, dv]), F),
                       output=view(0x5000000, Layout.c_contiguous([b, 1, h, dv]), F),
                       log_decay=buffer(0x4000000, h, F), lengths=None, state_in=None,
                       state_out=view(0x6000000, out, F, 300))
        assert (said is None) == once, (out, said)
        nested, reach = True, 1
        for s, n in sorted((abs(s), n) for s, n in zip(out.strides, out.shape) if n > 1):
            nested, reach = nested and s >= reach, reach + s * (n - 1)
        taken, refused, crossed = taken + once, refused + (not once), crossed + (once and not nested)
    assert taken > 500 and refused > 500 and crossed > 20


def test_views_too_tangled_to_decide_are_refused():
    """Strides that cross one another many times end in a refusal, and soon."""
    q = N([200, 1, 200, 200], [0, 0, 0, 1])
    first = N([200, 200, 200, 2], [2 * 999983, 2 * 999979, 2 * 999961, 1])
    last = N([200, 200, 200, 2], [80000, 400, 2, 1], 3)
    n = 2 * (999983 + 999979 + 999961) * 200
    said = refusal(attention, q=view(0x1000000, q, F, 200), k=view(0x2000000, q, F, 200),
                   v=view(0x3000000, N([200, 1, 200, 2], [0, 0, 0, 1]), F, 2),
                   output=view(0x5000000, Layout.c_contiguous([200, 1, 200, 2]), F), log_decay=buffer(0x4000000, 200, F),
                   lengths=None, state_in=view(0x10000000, first, F, n), state_out=view(0x10000000, last, F, n))
    assert said is None or "view of the state" in said


@pytest.mark.parametrize("call,at,what", [(norm, "residual", "residual"), (norm, "residual_out", "residual output"),
                                          (attention, "state_in", "attention state"),
                                          (attention, "state_out", "attention state output")])
def test_a_buffer_without_a_layout_is_refused(monkeypatch, call, at, what):
    """It would be left out without a word: h without the residual, an empty state."""
    from hephaestus_amd import layer_ops

    plain = layer_ops._view
    lost = view(0x9000000, Layout.c_contiguous([2]), F)
    monkeypatch.setattr(layer_ops, "_view", lambda v: (*plain(v)[:2], None) if v is lost else plain(v))
    monkeypatch.setattr(layer_ops, "_typed", lambda *_: None)
    assert refusal(call, **{at: lost}) == f"invalid configuration: {what} has a buffer and no layout"
