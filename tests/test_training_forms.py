"""That the sizes of the GPU tests reach every kernel of the training operators:
the rules are asked on the host (tests/cpp/training_forms.cpp)."""
from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest

import test_gpu_layer_norm as norm
import test_gpu_training_forms as forms

HERE = Path(__file__).resolve().parent
FORMS = HERE.parent / "hephaestus_amd" / "csrc" / "training_forms.hpp"
U64, I64, I32 = ctypes.c_uint64, ctypes.c_int64, ctypes.c_int32
SIZE = {"bf16": 2, "f32": 4}


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    path = tmp_path_factory.mktemp("rules") / "training_forms.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-o", str(path),
                    str(HERE / "cpp" / "training_forms.cpp")], check=True)
    lib = ctypes.CDLL(str(path))
    lib.norm_row.argtypes = [U64, U64]
    lib.recurrence_form.argtypes = [I32, I32, U64, U64, U64, U64, ctypes.POINTER(ctypes.c_uint32)]
    lib.product_form.argtypes = [U64, U64, U64, U64, ctypes.POINTER(U64)]
    lib.copies.argtypes = [U64, U64, I64, U64]
    lib.gradient_pieces.argtypes = [U64, U64, U64, U64, ctypes.POINTER(U64)]
    return lib


def names(enum):
    return re.findall(r"k\w+", re.search(rf"enum class {enum}[^{{]*\{{(.*?)\}}", FORMS.read_text(), re.S)[1])


def product(rules, m, n, k, size):
    form = (U64 * 3)()
    rules.product_form(m, n, k, size, form)
    return list(form)


def recurrence(rules, dtype, is_backward, size, at=0):
    form = (ctypes.c_uint32 * 4)()
    rules.recurrence_form(dtype == "f32", is_backward, *size, at, form)
    return list(form)


def test_every_tile_of_products_is_reached(rules):
    tiles = names("ProductTile")
    for dtype, by_tile in forms.TILES.items():
        assert list(by_tile) == tiles
        for place, tile in enumerate(tiles):
            for size in by_tile[tile]:
                assert product(rules, *size, SIZE[dtype])[:2] == [place, 1], (dtype, tile, size)
        for tile, sizes in forms.PARTS[dtype].items():
            for size in sizes:
                got = product(rules, *size, SIZE[dtype])
                assert got[0] == tiles.index(tile) and got[1] > 1, (dtype, tile, size, got)


def test_parts_of_products_hold_all_of_k(rules):
    for m, n in ((1, 1), (16, 2048), (300, 300), (8192, 4096)):
        for k in (0, 1, 63, 64, 1000, 32000, 130001):
            for size in (2, 4):
                _, parts, span = product(rules, m, n, k, size)
                assert span % (128 // size) == 0 and parts * span >= k and (parts - 1) * span < max(1, k), (m, n, k)


def test_every_recurrence_is_reached(rules):
    tiles = names("RecurrenceTile")
    reached = set()
    for form, sizes in forms.RECURRENCES.items():
        for size in sizes:
            for dtype in SIZE:
                for is_backward in (0, 1):
                    tile, parts, on_dwords, span = recurrence(rules, dtype, is_backward, size)
                    assert parts * span >= size[1] and (parts - 1) * span < size[1]
                    reached.add((dtype, is_backward, tiles[tile], parts > 1, dtype == "bf16" and on_dwords))
                    if form == "parts":
                        assert parts > 1
    for dtype in SIZE:
        for on_dwords in {dtype == "bf16", False}:
            for is_backward in (0, 1):
                kernels = [("kOne", False), ("kFew", False), ("kMany", False), ("kMany", True)]
                kernels += [] if is_backward else [("kLong", False)]
                for tile, parts in kernels:
                    assert (dtype, is_backward, tile, parts, on_dwords) in reached, (dtype, is_backward, tile, parts, on_dwords)
    # An operand off dwords is read by elements.
    assert recurrence(rules, "bf16", 0, (1, 1000, 130), at=2)[2] == 0


def test_every_row_of_norms_is_reached(rules):
    for size in SIZE.values():
        assert {rules.norm_row(cols, size) for _, cols in norm.WIDTHS} == set(range(len(names("NormRow"))))


def test_rows_that_are_copied(rules):
    """Off dwords, backwards or far apart; of the backward pass's weight also those that
    do not end with 16 bytes."""
    assert rules.copies(2, 0, 64, 64) == 0 and rules.copies(4, 0, 64, 64) == 0
    assert rules.copies(2, 2, 64, 64) == 3 and rules.copies(2, 0, 65, 64) == 3
    assert rules.copies(2, 0, -64, 64) == 3 and rules.copies(4, 0, -64, 64) == 3
    assert rules.copies(2, 0, 0, 64) == 0
    assert rules.copies(2, 0, 1 << 21, 64) == 0 and rules.copies(2, 0, (1 << 21) + 2, 64) == 3
    assert rules.copies(2, 0, 68, 60) == 2 and rules.copies(4, 0, 66, 66) == 2


def test_gradients_in_pieces(rules):
    form = (U64 * 2)()
    for size, rows in ((2, 70000), (4, 35000)):
        rules.gradient_pieces(size, rows, 4500, 8, form)
        assert form[0] == 3
        rules.gradient_pieces(size, 4, 4500, 8, form)
        assert form[0] == 1
    # G of a piece has at most 256 MiB, whatever the vocabulary.
    rules.gradient_pieces(2, 8192, 1 << 20, 64, form)
    assert form[1] <= (256 << 20) + (64 << 20)
