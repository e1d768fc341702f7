"""Which places of a gradient beside its logits are taken (credit_amd/csrc/
logits_rules.hpp, may_share): the logits themselves, memory apart from them, and
rows that lie between theirs.  Against sets of bytes.  No GPU."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

BASE = 1 << 20


@pytest.fixture(scope="module")
def may_share(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    source = Path(__file__).resolve().parent / "cpp" / "logits_overlap_query.cpp"
    out = tmp_path_factory.mktemp("overlap") / "logits_overlap.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", str(source), "-o",
                    str(out)], check=True)
    fn = ctypes.CDLL(str(out)).logits_may_share
    i64, ptr = ctypes.c_int64, ctypes.c_size_t
    fn.argtypes, fn.restype = [ptr, i64, ptr, i64, i64, i64, ptr], ctypes.c_int
    return fn


def elements(at, ld, rows, cols):
    return {at + r * ld + c for r in range(rows) for c in range(cols)}


@pytest.mark.parametrize("elem", [2, 4])
def test_against_sets(may_share, elem):
    for rows in (1, 2, 3):
        for cols in (1, 3, 4):
            for ld in range(cols, 10):
                for ldb in {ld, cols, 9}:
                    mine = elements(0, ld, rows, cols)
                    for off in range(-34, 35):
                        got = may_share(BASE, ld, BASE + off * elem, ldb, rows, cols, elem)
                        same = off == 0 and (rows == 1 or ld == ldb)
                        apart = not mine & elements(off, ldb, rows, cols)
                        if same:
                            assert got
                        elif got:
                            assert apart, (rows, cols, ld, ldb, off)
                        elif apart:
                            # Refused although apart: between rows of another distance alone.
                            assert ld != ldb and rows > 1, (rows, cols, ld, off)


def test_halves_of_one_buffer(may_share):
    for cols, ld in ((50001, 100002), (128, 256), (7, 30)):
        for elem in (2, 4):
            for rows in (2, 1000):
                for sign in (1, -1):
                    assert may_share(BASE << 20, ld, (BASE << 20) + sign * cols * elem, ld, rows,
                                     cols, elem)
                    assert not may_share(BASE << 20, ld, (BASE << 20) + sign * (cols - 1) * elem,
                                         ld, rows, cols, elem)
