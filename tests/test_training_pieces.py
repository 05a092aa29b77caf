"""That the sizes of the GPU tests reach grad_x of pieces of the vocabulary in parts and
without, in either type."""
from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest

import test_gpu_cross_entropy_pieces as pieces
from test_training_forms import SIZE, U64, product, rules  # noqa: F401 (a fixture)

HERE = Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def gradient_piece(tmp_path_factory):
    path = tmp_path_factory.mktemp("rules") / "training_launches.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-o", str(path),
                    str(HERE / "cpp" / "training_launches.cpp")], check=True)
    fn = ctypes.CDLL(str(path)).gradient_piece
    fn.argtypes = [U64, U64, U64, U64, ctypes.POINTER(U64)]

    def ask(*size):
        form = (U64 * 3)()
        fn(*size, form)
        return list(form)

    return ask


@pytest.mark.parametrize("is_cut", [True, False])
def test_sizes_reach_their_forms(rules, gradient_piece, is_cut):  # noqa: F811
    sizes = pieces.PARTS if is_cut else pieces.WHOLE
    assert {dtype for dtype, *_ in sizes} == set(SIZE)
    for dtype, rows, vocab, width in sizes:
        piece = gradient_piece(SIZE[dtype], rows, vocab, width)[0]
        words = [min(piece, vocab - first) for first in range(0, vocab, piece)]
        assert len(words) >= 2
        for n in words:
            assert (product(rules, rows, width, n, SIZE[dtype])[1] > 1) == is_cut, (dtype, n)
