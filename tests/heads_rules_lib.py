"""The host rules of the operators on heads (credit_amd/csrc/heads_rules.hpp,
attention_rules.hpp), built with g++ for tests that ask which way a call goes."""
import ctypes
import subprocess
from pathlib import Path

FEW, MANY = 32, 128  # rows of a small and of a large tile


def build(folder) -> ctypes.CDLL:
    source = Path(__file__).resolve().parent / "cpp" / "heads_rules_query.cpp"
    out = Path(folder) / "heads_rules.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", str(source), "-o", str(out)],
                   check=True)
    lib = ctypes.CDLL(str(out))
    i64, i32 = ctypes.c_int64, ctypes.c_int
    lib.attention_tile_rows.argtypes = [i64] * 4 + [i32, i64]
    lib.attention_units.argtypes = [i64] * 4 + [i32, i64, i64]
    return lib


def way(rules, args, window=0) -> tuple[int, bool]:
    """Rows of a tile, and whether there are parts, of hip_lib.paged_attention(*args)."""
    q, k, table = args[0], args[1], args[3]
    shape = (q.shape[0], table.shape[0], q.shape[1], k.shape[2], q.shape[2],
             table.shape[1] * k.shape[1])
    return rules.attention_tile_rows(*shape), rules.attention_units(*shape, window) > 0
