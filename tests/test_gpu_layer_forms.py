"""Every kernel of the layer operators, at sizes that reach it (that they do is
tested in test_layer_forms.py, on the host), against plain forms in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

import hephaestus_amd as hx
import test_gpu_layer_streams as streams
from layer_reference import EPS16, EPS32, as_float64
from test_gpu_linear_attention import TYPES
from test_gpu_linear_attention import check as check_attention
from test_gpu_linear_attention import operands as attention_operands
from test_gpu_linear_attention import run as run_attention
from test_gpu_matmul_i8 import operands as matmul_operands
from test_gpu_matmul_i8 import run as run_matmul

pytestmark = pytest.mark.gpu

# Sizes (m, n, k) of each tile, with a whole number of steps of k and not, m and
# n off the tile.  Those of 4096 bytes and more of k are the forms for long rows.
TILES = {
    "k256x256": [(3300, 3300, 200), (3290, 3310, 256)],
    "k128x128Pairs": [(2100, 2100, 300), (2090, 2110, 640)],
    "k128x128": [(1800, 1850, 260), (1790, 1810, 512)],
    "k96x96": [(1400, 1400, 4100), (1380, 1390, 4608)],
    "k64x64Groups": [(128, 5200, 4100), (130, 5190, 4224)],
    "k64x64": [(700, 1000, 500), (690, 1010, 128)],
    "k64x32Pairs": [(64, 8220, 384), (60, 8230, 516)],
    "k64x32": [(60, 6000, 516), (63, 6010, 1280)],
    "k32x32Pairs": [(40, 4300, 640), (39, 4310, 516)],
    "k32x32": [(40, 2600, 516), (38, 2590, 1024)],
    "k32x16": [(40, 100, 1500), (37, 90, 2048)],
}
# Of each form for few tokens, and where its rows begin (bytes past a dword).
FEW_TOKENS = {
    "16": [(1, 100, 300, 0), (16, 1000, 1280, 0)],
    "16 wide": [(1, 8200, 300, 0), (13, 8230, 2048, 0)],
    "16 bytes": [(16, 100, 301, 0), (5, 1000, 1280, 1)],
    "16 wide bytes": [(16, 8200, 301, 0), (2, 8230, 1155, 3)],
    "32 bytes": [(20, 100, 301, 0), (32, 1000, 1280, 2)],
    "32 wide bytes": [(20, 8200, 301, 0), (31, 8230, 1155, 1)],
}
# Widths of each kernel for prompts; both are multiples of 8, for loads without registers.
WIDTHS = [(64, 64), (96, 64), (128, 64), (256, 64), (64, 128), (96, 80), (128, 72), (128, 128), (200, 136)]
ODD_WIDTHS = [(37, 53), (90, 61), (101, 49), (180, 50), (50, 77), (90, 90), (127, 129)]
# Batch, heads and chunks of prompts whose blocks take all of one, and of prompts that are
# cut into parts of several chunks.
WHOLE = (2, 130, 5)
CUT = (2, 16, 20)
# Batch, heads, dk and dv of states that the caches do not keep.
STREAMED = [(64, 65, 32, 130), (65, 64, 64, 66), (33, 32, 128, 128), (17, 32, 256, 128), (130, 70, 37, 53)]
CHUNK = {"f32": 32, "bf16": 64}


def check_matmul(a, b, sa, sb, got):
    total = a.astype(np.float64) @ b.astype(np.float64).T  # exact: sums below 2^53
    want = sa.astype(np.float64)[:, None] * total * sb.astype(np.float64)
    # The sum as f32, two products, and the output's own rounding.
    bound = 4 * EPS32 + (EPS16 if got.dtype == hx.bfloat16 else 0)
    assert np.all(np.abs(as_float64(got) - want) <= np.abs(want) * bound)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("m,n,k", [size for sizes in TILES.values() for size in sizes])
def test_products_of_every_tile(device, dtype, pad, m, n, k):
    """With rows on dwords, and on none of the same address modulo 4: these are copied first."""
    ops = matmul_operands(m, n, k, 51)
    check_matmul(*ops, run_matmul(device, *ops, TYPES[dtype], pad=pad, offset=pad))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k,offset", [size for sizes in FEW_TOKENS.values() for size in sizes])
def test_products_of_few_tokens(device, dtype, m, n, k, offset):
    ops = matmul_operands(m, n, k, 52)
    check_matmul(*ops, run_matmul(device, *ops, TYPES[dtype], offset=offset, prepared=True))


def by_pairs(q, k, v, log_decay, scale, state):
    """One head's outputs and last state from every token's pair with those before
    it, in 64 bits, and both with every term's magnitude."""
    q, k, v, g, state = as_float64(q), as_float64(k), as_float64(v), float(log_decay), state.astype(np.float64)
    at = np.arange(len(q), dtype=np.float64)
    far = at[:, None] - at
    within = np.exp(g * np.maximum(far, 0)) * (far >= 0)
    since = np.exp(g * (at + 1))[:, None]
    left = np.exp(g * (len(q) - 1 - at))[:, None]

    def outputs(q, k, v, state):
        return ((q @ k.T) * within) @ v + since * (q @ state), (k * left).T @ v + since[-1] * state

    out, last = outputs(q, k, v, state)
    size, last_size = outputs(*(np.abs(x) for x in (q, k, v, state)))
    return scale * out, last, scale * size, last_size


def check_prompt(q, k, v, decay, state, lengths, got, chunk, heads):
    scale = float(np.float32(q.shape[3] ** -0.5))
    group = q.shape[2] // k.shape[2]
    for b, h in heads:
        n = q.shape[1] if lengths is None else lengths[b]
        want, last, size, last_size = by_pairs(q[b, :n, h], k[b, :n, h // group], v[b, :n, h // group], decay[h], scale,
                                               state[b, h])
        # For each chunk the state's decay and sum, and as much where parts are
        # joined; the sums over a chunk and over dk; some for weights and scale.
        state_steps = (4 * -(-n // chunk) + chunk + 32) * EPS32
        inner = state_steps + q.shape[3] * EPS32
        bound = inner * size
        if q.dtype == hx.bfloat16:  # two bf16 terms a score and an element of the state; the output's rounding
            inner += 2 * 2.0**-15
            bound = inner * size + EPS16 * (np.abs(want) + inner * size)
        off = np.abs(as_float64(got[0][b, :n, h]) - want)
        assert np.all(off <= bound), (b, h, np.unravel_index(np.argmax(off - bound), off.shape))
        off = np.abs(got[1][b, h] - last)
        assert np.all(off <= state_steps * last_size), (b, h, np.unravel_index(np.argmax(off), off.shape))
        assert not as_float64(got[0][b, n:, h]).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("prompt", [WHOLE, CUT], ids=["whole", "cut"])
@pytest.mark.parametrize("dk,dv", WIDTHS + ODD_WIDTHS)
def test_prompts_of_every_kernel(device, dtype, offset, prompt, dk, dv):
    """Rows that are loaded without registers, and at an odd element, which are
    not; a sequence that ends within a chunk and a part, one that fills both."""
    batch, heads, chunks = prompt
    tokens = chunks * CHUNK[dtype]
    lengths = [tokens, tokens * 2 // 3 + 5]
    ops = attention_operands(TYPES[dtype], batch, tokens, heads, 2, dk, dv, 53)
    got = run_attention(device, *ops, lengths, offset=offset, prepared=True)
    check_prompt(*ops, lengths, got, CHUNK[dtype], [(0, 0), (0, heads - 1), (1, heads // 2)])


@pytest.mark.parametrize("dtype", TYPES)
def test_many_chunks_in_a_block(device, dtype):
    ops = attention_operands(TYPES[dtype], 1, 40 * CHUNK[dtype] + 1, 520, 520, 16, 24, 54)
    check_prompt(*ops, None, run_attention(device, *ops), CHUNK[dtype], [(0, 0), (0, 300), (0, 519)])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 3])
@pytest.mark.parametrize("batch,heads,dk,dv", STREAMED)
def test_states_beyond_the_caches(device, dtype, tokens, batch, heads, dk, dv):
    """All written; every 37th sequence is compared, and the last."""
    q, k, v, decay, state = attention_operands(TYPES[dtype], batch, tokens, heads, heads, dk, dv, 55)
    got, last = run_attention(device, q, k, v, decay, state)
    some = sorted({*range(0, batch, 37), batch - 1})
    check_attention(*(x[some] for x in (q, k, v)), decay, state[some], None, (got[some], last[some]))
    assert np.isfinite(last).all() and not (last == 5).all(axis=(2, 3)).any()


class WorkspaceLayer(streams.Layer):
    """The norm, a product whose rows are copied first and a prompt that is cut:
    both keep what they hold between launches in a workspace."""

    def __init__(self, device):
        super().__init__(device)
        del self.cases[1:]
        self.add_matmul(70, 300, 385)
        self.add_attention(2500)
        for _, _, plan, *_ in self.cases[1:]:
            assert plan.workspace_bytes() > 0


@pytest.fixture(scope="module")
def workspaces(device):
    return WorkspaceLayer(device)


@pytest.mark.parametrize("use", [streams.test_plans_read_their_operands_anew,
                                 streams.test_immediate_calls_on_a_callers_stream, streams.test_plans_under_capture,
                                 streams.test_immediate_calls_that_take_scratch_refuse_capture],
                         ids=lambda f: f.__name__[5:])
def test_workspaces(device, workspaces, use):
    use(device, workspaces)


def test_two_streams_do_not_share_scratch(device):
    """Immediate calls on two streams at once, each with its own scratch."""
    layers = [WorkspaceLayer(device) for _ in range(2)]
    ins = [layer.write(60 + i) for i, layer in enumerate(layers)]
    queues = [streams.Stream() for _ in layers]
    try:
        for _ in range(4):
            for layer, queue in zip(layers, queues):
                for _, _, _, call, _ in layer.cases:
                    call(queue.value)
        for queue in queues:
            queue.sync()
        for layer, x in zip(layers, ins):
            layer.verify(x)
    finally:
        for queue in queues:
            queue.close(device)
