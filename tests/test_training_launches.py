"""Products of more tiles than a launch has blocks: the rule is asked on the host, and the
kernel's order of tiles is followed."""
from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    path = tmp_path_factory.mktemp("rules") / "training_launches.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-o", str(path),
                    str(HERE / "cpp" / "training_launches.cpp")], check=True)
    fn = ctypes.CDLL(str(path)).tiles_of_a_launch
    fn.argtypes, fn.restype = [ctypes.c_uint64], ctypes.c_uint64
    return fn


@pytest.mark.parametrize("threads", [256, 512])
def test_a_launch_has_fewer_than_32_bits_of_threads(rule, threads):
    most = rule(threads)
    assert most * threads < 1 << 32 and most % 8 == 0
    assert (most + 8) * threads >= 1 << 32  # and no fewer than it may


@pytest.mark.parametrize("total,most", [(1, 16), (7, 16), (16, 16), (17, 16), (101, 16), (100, 104)])
def test_every_tile_is_taken_once(total, most):
    """Blocks go to the eight XCDs in turn, each of which takes a run of the launch's."""
    seen = []
    for first in range(0, total, most):
        blocks = min(most, total - first)
        share, rest = blocks // 8, blocks % 8
        seen += [first + b % 8 * share + min(b % 8, rest) + b // 8 for b in range(blocks)]
    assert sorted(seen) == list(range(total))
