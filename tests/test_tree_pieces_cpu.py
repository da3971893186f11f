"""What the merge of a cut tree item may read, compiled for the host: entries that no CTA wrote (its bounded wait gave up)
hold anything, and name nothing outside the workspace."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "infera_b200" / "csrc"
SOURCE = """
#include "tree_pieces.h"
extern "C" int exist(int first, int count, int runs) { return ib200::pieces_exist(first, count, runs); }
extern "C" long long at(int first, int k) { return ib200::piece_at(first, k); }
"""
ANY = [-(2 ** 31), -(2 ** 31) + 1, -65536, -2, -1, 0, 1, 2, 3, 36, 37, 38, 295, 296, 297, 65535, 2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("pieces")
    (d / "p.cpp").write_text(SOURCE)
    # -ftrapv: a sum that passes 32 bits ends the test
    subprocess.run([gxx, "-O1", "-ftrapv", "-shared", "-fPIC", "-I", str(CSRC), str(d / "p.cpp"), "-o", str(d / "p.so")], check=True)
    lib = ctypes.CDLL(str(d / "p.so"))
    lib.at.restype = ctypes.c_longlong
    return lib


@pytest.mark.parametrize("runs", [1, 2, 37, 296, 65535])
def test_only_pieces_of_the_runs_are_read(lib, runs):
    for first in ANY:
        for count in ANY:
            inside = 0 <= first <= first + count <= runs and count >= 0
            assert bool(lib.exist(first, count, runs)) == inside, (first, count)
            if inside and count:  # the workspace has two places a run
                places = [lib.at(first, k) for k in {0, count // 2, count - 1}]
                assert all(0 <= p < 2 * runs for p in places)


def test_pieces_lie_in_places_of_their_own(lib):
    # an item that begins in run 4 and the one before it, which ends there
    assert lib.at(4, 0) == 9 and lib.at(2, 2) == 8 and lib.at(0, 0) == 1 and lib.at(0, 1) == 2
