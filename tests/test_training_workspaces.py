"""The workspaces that include/hx.h states for the training operators, by the rules that
size them."""
from __future__ import annotations

import ctypes
import itertools
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent
U64 = ctypes.c_uint64


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    path = tmp_path_factory.mktemp("rules") / "training_launches.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-o", str(path),
                    str(HERE / "cpp" / "training_launches.cpp")], check=True)
    lib = ctypes.CDLL(str(path))
    lib.gradient_piece.argtypes = [U64, U64, U64, U64, ctypes.POINTER(U64)]
    lib.norm_runs.argtypes, lib.norm_runs.restype = [U64, U64, U64], U64
    lib.map_bytes.argtypes, lib.map_bytes.restype = [U64, ctypes.c_int, U64, U64, U64], U64
    return lib


def test_gradients_of_logits(lib):
    """At most 256 MiB or 256 words of every row, whatever the rows and the vocabulary."""
    form = (U64 * 3)()
    for size, rows, vocab in itertools.product((2, 4), (1, 1000, 8192, 300000, 1000000, 1 << 24, (1 << 28) - 1),
                                               (1, 255, 1000, 131072, 1 << 20, (1 << 28) - 1)):
        lib.gradient_piece(size, rows, vocab, 64, form)
        assert form[0] >= 256 and form[0] % 256 == 0
        assert form[1] <= max(256 << 20, rows * 256 * size), (size, rows, vocab)
    lib.gradient_piece(2, 1000000, 1000, 64, form)
    assert form[1] == 1000000 * 256 * 2  # 488 MiB


def test_runs_of_rows_of_norms(lib):
    for size, rows, cols in itertools.product((2, 4), (1, 3, 100, 512, 1000, 16384, 1 << 20, (1 << 31) - 1),
                                              (1, 64, 1000, 2048, 8192, 20000, 1 << 20)):
        assert 1 <= lib.norm_runs(size, rows, cols) <= min(rows, 512), (size, rows, cols)


def test_maps_of_parts(lib):
    most = 0
    for vector, is_backward, batch, tokens, channels in itertools.product(
            (1, 2), (0, 1), (1, 2, 5, 64, 159, 160), (1, 33, 128, 193, 1000, 65536, 1 << 20),
            (2, 64, 96, 128, 1024, 1600, 4096, 20000)):
        most = max(most, lib.map_bytes(vector, is_backward, batch, tokens, channels))
    assert 0 < most <= 512 << 10
