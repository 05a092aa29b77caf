"""That the sizes of the GPU tests reach every kernel of the layer operators: the
rules are asked on the host (tests/cpp/layer_forms.cpp)."""
from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest

import test_gpu_layer_forms as forms
import test_gpu_norm_tiny_rows as tiny

HERE = Path(__file__).resolve().parent
CSRC = HERE.parent / "hephaestus_amd" / "csrc"
U64, I64 = ctypes.c_uint64, ctypes.c_int64


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    path = tmp_path_factory.mktemp("rules") / "layer_forms.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-o", str(path),
                    str(HERE / "cpp" / "layer_forms.cpp")], check=True)
    lib = ctypes.CDLL(str(path))
    lib.matmul_form.argtypes = [U64] * 5 + [I64] * 2
    lib.attention_form.argtypes = [ctypes.c_int32] + [U64] * 6 + [ctypes.POINTER(ctypes.c_uint32)]
    return lib


def tile_names():
    text = (CSRC / "layer_forms.hpp").read_text()
    return re.findall(r"k\d+x\d+\w*", re.search(r"enum class MatmulTile[^{]*\{(.*?)\}", text, re.S)[1])


def attention_form(rules, dtype, batch, tokens, heads, dk, dv, at=0):
    form = (ctypes.c_uint32 * 6)()
    rules.attention_form(dtype == "f32", batch, tokens, heads, dk, dv, at, form)
    return list(form)


def test_every_tile_of_products_is_reached(rules):
    names = tile_names()
    assert list(forms.TILES) == names
    for place, name in enumerate(names):
        for m, n, k in forms.TILES[name]:
            assert rules.matmul_form(m, n, k, 0x1000, 0x2000, k, k) == place, (name, m, n, k)
            # pad = offset = 1, and b one more apart
            assert rules.matmul_form(m, n, k, 0x1001, 0x2001, k + 1, k + 2) == 1000 + place, (name, m, n, k)
        assert {k % 128 == 0 for _, _, k in forms.TILES[name]} == {False, True}


def test_every_form_for_few_tokens_is_reached(rules):
    for name, sizes in forms.FEW_TOKENS.items():
        want = 100 + 4 * ("32" in name) + 2 * ("wide" in name) + ("bytes" not in name)
        for m, n, k, offset in sizes:
            assert rules.matmul_form(m, n, k, 0x1000 + offset, 0x2000 + offset, k, k) == want, (name, m, n, k)


def test_every_kernel_for_prompts_is_reached(rules):
    def kernel(dk, waves):
        return min(w for w in (64, 96, 128, 256) if dk <= w), waves

    for dtype, size in (("f32", 4), ("bf16", 2)):
        for prompt, cut in ((forms.WHOLE, False), (forms.CUT, True)):
            batch, heads, chunks = prompt
            reached = set()
            for dk, dv in forms.WIDTHS + forms.ODD_WIDTHS:
                for offset in (0, 1):
                    by_chunks, _, waves, direct, parts, span = attention_form(
                        rules, dtype, batch, chunks * forms.CHUNK[dtype], heads, dk, dv, offset * size)
                    assert by_chunks and (parts > 1) == cut and (span > 1 or not cut), (dtype, dk, dv, parts, span)
                    reached.add((*kernel(dk, waves), bool(direct)))
                assert (dv % 4 == 0) == ((dk, dv) in forms.WIDTHS)  # both ways of joining
            assert reached == {(w, n, d) for w, n in ((64, 4), (96, 4), (128, 4), (256, 4), (64, 8), (96, 8), (128, 8))
                               for d in (False, True)}, (dtype, cut)
        by_chunks, _, _, _, parts, span = attention_form(rules, dtype, 1, 40 * forms.CHUNK[dtype] + 1, 520, 16, 24)
        assert by_chunks and parts == 1 and span == 41


def test_every_kernel_for_single_tokens_is_reached(rules):
    reached = set()
    for batch, heads, dk, dv in forms.STREAMED:
        for tokens in (1, 3):
            for dtype in ("f32", "bf16"):
                by_chunks, streamed, *_ = attention_form(rules, dtype, batch, tokens, heads, dk, dv)
                assert not by_chunks and streamed
        reached.add(min(w for w in (32, 64, 128, 256) if dk <= w))
    assert reached == {32, 64, 128, 256}


def test_every_width_of_norms_is_reached():
    """Vectors of a row at which norm_quantize.hip goes to another kernel."""
    text = (CSRC / "norm_quantize.hip").read_text()
    bounds = [int(n) for n in re.findall(r"if \(vectors <= (\d+)\) run", text)]
    assert len(bounds) == 8
    for elements in (4, 8):
        reached = {sum(-(-cols // elements) > b for b in bounds) for cols in tiny.COLS}
        assert reached == set(range(9))


def test_wide_heads_are_not_cut_too_early(rules):
    """A block has at most 128 columns of v, whatever the head: its chunks take no longer."""
    for dtype, tokens, heads, dk, dv in (("bf16", 256, 8, 128, 2048), ("bf16", 192, 8, 128, 1024),
                                         ("bf16", 256, 8, 256, 1024), ("bf16", 128, 4, 256, 1024),
                                         ("f32", 64, 8, 128, 2048)):
        assert attention_form(rules, dtype, 1, tokens, heads, dk, dv)[4] == 1
    for dtype, tokens, heads, dk, dv, parts in (("bf16", 1024, 8, 128, 512, 8), ("bf16", 640, 32, 128, 256, 4),
                                                ("f32", 512, 8, 128, 512, 8)):
        assert attention_form(rules, dtype, 1, tokens, heads, dk, dv)[4] == parts


def test_the_prompt_under_capture_is_cut(rules):
    """The one of tests/test_gpu_layer_streams.py, and the longer one with workspaces."""
    assert attention_form(rules, "bf16", 1, 300, 2, 64, 48)[4] > 1
    assert attention_form(rules, "bf16", 1, 2500, 2, 64, 48)[4] > 1
