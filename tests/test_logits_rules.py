"""How the forwards of the operators on logits cut rows into parts, and the
workspace they ask for (credit_amd/csrc/logits_rules.hpp).  No GPU."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

from credit_amd import hip_lib

I64 = ctypes.c_int64
BATCH, MOST_PARTS, MOST_ROWS = 8192, 64, 1024


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    source = Path(__file__).resolve().parent / "cpp" / "logits_rules_query.cpp"
    out = tmp_path_factory.mktemp("rules") / "logits_rules.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", str(source), "-o",
                    str(out)], check=True)
    lib = ctypes.CDLL(str(out))
    lib.logits_auto_parts.argtypes, lib.logits_auto_parts.restype = [I64, I64, ctypes.c_int], I64
    lib.logits_workspace.argtypes = [I64, I64, ctypes.c_int, I64, ctypes.c_int]
    lib.logits_parts_bytes.argtypes = [I64, I64, I64, ctypes.c_int]
    lib.logits_workspace.restype = lib.logits_parts_bytes.restype = ctypes.c_size_t
    return lib


def test_only_few_wide_rows_are_cut(rules):
    for top in (0, 1):
        for rows in (257, 512, 4096, 1 << 30):
            assert rules.logits_auto_parts(rows, 32, top) == 1
        for rows in (1, 16, 256):
            for batches in (1, 2, 3):
                assert rules.logits_auto_parts(rows, batches, top) == 1
    assert rules.logits_auto_parts(1, 16, 0) == rules.logits_auto_parts(1, 16, 1) == 16
    assert rules.logits_auto_parts(1, 4, 1) == 1
    assert rules.logits_auto_parts(64, 16, 0) == 4
    assert rules.logits_auto_parts(128, 16, 0) == 2 and rules.logits_auto_parts(128, 16, 1) == 1
    assert rules.logits_auto_parts(1, 1 << 16, 0) == MOST_PARTS


def test_the_workspace_covers_every_type_alignment_and_plan(rules):
    for rows in (1, 3, 64, 100, 1024, 1025):
        for cols in (1, 8191, 8192, 8193, 50001, 65530, 65536, 131072, 262144, 1 << 22):
            for split in (0, 1, 2, 5, 64):
                for alternatives in (0, 1):
                    have = rules.logits_workspace(rows, cols, 0, split, alternatives)
                    for slack in (0, 3, 31, 63):
                        batches = (cols + slack + BATCH - 1) // BATCH
                        for top in range(alternatives + 1):
                            want = split or rules.logits_auto_parts(rows, batches, top)
                            each = -(-batches // want)
                            n = -(-batches // each)
                            if n >= 2 and rows <= MOST_ROWS:
                                assert n * each >= batches and n <= MOST_PARTS
                                assert have >= rules.logits_parts_bytes(rows, n, each, top)
            assert rules.logits_workspace(rows, cols, 1, 0, 1) == 0


def test_workspace_bytes_of_the_library(lib):
    for op in ("token_logprob_fwd", "topk_distill_fwd"):
        assert hip_lib.workspace_bytes(op, 4096, 131072) == 0
        assert hip_lib.workspace_bytes(op, 8, 131072, "read") == 0
        # Header, counters and slots, then what the parts leave.
        assert hip_lib.workspace_bytes(op, 8, 131072) > (5 << 20) + 256
    assert (hip_lib.workspace_bytes("token_logprob_fwd", 8, 131072, "split", 2)
            > hip_lib.workspace_bytes("topk_distill_fwd", 8, 131072, "split", 2))
    for op in ("token_logprob_bwd", "topk_distill_bwd"):
        assert hip_lib.workspace_bytes(op, 8, 131072) == 0
