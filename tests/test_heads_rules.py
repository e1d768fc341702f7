"""Where tensors of the operators on heads may lie, how heads are dealt to groups of
lanes and attention to workgroups (credit_amd/csrc/heads_rules.hpp,
attention_rules.hpp).  No GPU."""
import ctypes
import random
import shutil
import subprocess
from pathlib import Path

import pytest

from credit_amd import hip_lib

I64, INT, SIZE = ctypes.c_int64, ctypes.c_int, ctypes.c_size_t
FEW, MANY, RESIDENT = 32, 128, 512


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    source = Path(__file__).resolve().parent / "cpp" / "heads_rules_query.cpp"
    out = tmp_path_factory.mktemp("rules") / "heads_rules.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", str(source), "-o",
                    str(out)], check=True)
    lib = ctypes.CDLL(str(out))
    place = I64 * 6
    for name, args, result in (
            ("heads_apart", [place, place], INT), ("heads_apart_within", [place], INT),
            ("heads_same", [place, place], INT), ("heads_run_of", [I64, I64, INT, INT, INT], INT),
            ("heads_groups_of", [INT, INT], INT),
            ("attention_tile_rows", [I64] * 4 + [INT, I64], INT), ("attention_tiles", [I64] * 3 + [INT], I64),
            ("attention_units", [I64] * 4 + [INT, I64, I64], INT),
            ("attention_workspace", [I64] * 4 + [INT, I64, I64], SIZE),
            ("attention_padded_dim", [INT], INT),
            ("attention_divide", [ctypes.c_uint32] * 2, ctypes.c_uint32)):
        fn = getattr(lib, name)
        fn.argtypes, fn.restype = args, result
    lib.place = place
    return lib


def touched(p):
    at, run, step, outer, count, width = p
    return [set(range(at + o * run + c * step, at + o * run + c * step + width))
            for o in range(outer) for c in range(count)]


def test_places_apart_share_no_byte(rules):
    """What is called apart is, over places small enough to count; the layouts that
    calls have are called so."""
    rng = random.Random(0)
    found = within = 0
    for _ in range(20000):
        ps = [(1000 + rng.randrange(60), rng.randrange(0, 40), rng.randrange(0, 20),
               rng.randrange(1, 4), rng.randrange(1, 4), rng.randrange(1, 8)) for _ in "ab"]
        if rng.random() < 0.5:
            ps[1] = (ps[1][0], *ps[0][1:3], *ps[1][3:])
        a, b = (rules.place(*p) for p in ps)
        bytes_a, bytes_b = (set().union(*touched(p)) for p in ps)
        if rules.heads_apart(a, b):
            found += 1
            assert not bytes_a & bytes_b, ps
        if rules.heads_apart_within(a):
            within += 1
            assert len(bytes_a) == sum(map(len, touched(ps[0]))), ps[0]
        assert rules.heads_apart(a, b) == rules.heads_apart(b, a)
    assert found > 1000 and within > 1000
    # Queries and keys as columns of one projection, heads first, and one behind the other.
    wide = (0, 96, 16, 5, 4, 16), (64, 96, 16, 5, 2, 16)
    first = (0, 16, 80, 5, 4, 16), (320, 16, 80, 5, 2, 16)
    for a, b in (wide, first):
        a, b = rules.place(*a), rules.place(*b)
        assert rules.heads_apart(a, b) and not rules.heads_apart(a, a)
        assert rules.heads_same(a, a) and not rules.heads_same(a, b)
        assert rules.heads_apart_within(a)
    # Tensors without elements.
    assert rules.heads_apart(rules.place(0, 1, 1, 0, 1, 1), rules.place(0, 1, 1, 1, 1, 1))


def test_groups_cover_the_heads(rules):
    for most in (1, 2, 4):
        for tokens in (1, 64, 1000, 4096, 1 << 20, 1 << 40):
            for lanes in (4, 8, 64):
                assert rules.heads_run_of(tokens, 40, 32, lanes, most) in (1, 2, 4)[:most]
        for n in (1, 2, 3, 8, 14, 32, 127, 1000):
            groups = rules.heads_groups_of(n, most)
            assert groups & (groups - 1) == 0 and groups * most >= n
            assert groups == 1 or groups // 2 * most < n
    assert rules.heads_run_of(1, 48, 32, 8, 4) == 1  # a token's heads side by side
    assert rules.heads_run_of(8192, 48, 32, 8, 4) == 4
    assert rules.heads_run_of(16384, 40, 32, 8, 2) == 2
    assert rules.heads_run_of(1 << 20, 3, 2, 8, 4) == 2  # no more than there are


def test_tiles_hold_every_sequence(rules):
    """A sequence's slots: from floor(first row / rows) + its number on, as many as its
    rows fill, below the next one's and the launch's."""
    rng = random.Random(1)
    for _ in range(2000):
        batch, group = rng.randrange(1, 9), rng.choice((1, 2, 5, 7, 8, 16))
        lengths = [rng.choice((0, 1, rng.randrange(70), rng.randrange(400)))
                   for _ in range(batch)]
        lead, tail = rng.randrange(40), rng.randrange(40)
        tokens = lead + sum(lengths) + tail
        rows = rules.attention_tile_rows(tokens, batch, group, 1, 128, rng.choice((100, 9000)))
        assert rows in (FEW, MANY)
        at, free = lead, 0
        for b, n in enumerate(lengths):
            first = at * group // rows + b
            assert first >= free
            free = first + -(-n * group // rows)
            at += n
        assert free <= rules.attention_tiles(tokens, batch, group, rows)


def test_tile_rows(rules):
    rows = rules.attention_tile_rows
    assert rows(64, 64, 32, 8, 128, 8192) == rows(8, 1, 32, 8, 128, 8192) == FEW
    assert rows(9, 1, 32, 8, 128, 8192) == MANY  # 36 rows over many positions
    assert rows(9, 1, 32, 8, 128, 2048) == FEW and rows(9, 1, 32, 8, 128, 2049) == MANY
    assert rows(248, 1, 32, 8, 128, 2048) == FEW and rows(256, 1, 32, 8, 128, 2048) == MANY
    assert rows(8192, 1, 16, 4, 200, 8192) == FEW and rows(8192, 1, 16, 4, 192, 8192) == MANY


def test_parts(rules):
    # Short sequences, long prompts and too many sequences to count through: whole tiles.
    units, workspace = rules.attention_units, rules.attention_workspace
    assert units(1, 1, 32, 8, 128, 512, 0) == 0
    assert units(8192, 1, 32, 8, 128, 8192, 0) == units(8192, 1, 32, 8, 256, 8192, 0) == 0
    assert units(2000, 2000, 32, 8, 128, 8192, 0) == 0
    assert units(1, 1, 32, 8, 128, 8192, 0) == 32  # 1 tile of 256 steps, 8 each
    assert units(1, 1, 32, 8, 128, 8192, 100) == 0  # 6 steps
    assert units(512, 1, 32, 8, 128, 8192, 0) == 64  # 17 tiles of 128 steps
    assert units(40, 1, 32, 8, 128, 8192, 0) == 32  # 2 of 128, one unit a CU
    assert units(40, 4, 8, 8, 128, 3000, 0) == 59  # 5 small tiles of 94
    assert units(33, 1, 8, 8, 128, 3000, 0) == 12  # 1 large one of 47, 4 each
    for heads, kv in ((32, 8), (8, 1), (14, 2), (64, 64), (1024, 1024), (600, 600)):
        for tokens, batch in ((1, 1), (64, 64), (512, 1), (300, 7), (40, 1)):
            for positions in (1, 300, 2048, 8192, 1 << 20, 1 << 30):
                for dim in (128, 256):
                    n = units(tokens, batch, heads, kv, dim, positions, 0)
                    assert n * kv <= max(RESIDENT, kv)
                    size = workspace(tokens, batch, heads, kv, dim, positions, 0)
                    # Two places a unit, offsets within 32 bits.
                    assert (size == 0) == (n == 0) and size < 1 << 31
                    # What is asked for without a window serves with any.
                    for window in (1, 100, 1000, 5000, 1 << 30):
                        assert size >= workspace(tokens, batch, heads, kv, dim, positions, window)


def test_divisors(rules):
    rng = random.Random(2)
    for d in [*range(1, 70), 96, 127, 128, 129, 1000, 4096, 65535, (1 << 20) + 1, (1 << 30)]:
        for n in [0, 1, d - 1, d, d + 1, 2 * d - 1, (1 << 31) - 1, (1 << 31) - d,
                  *(rng.randrange(1 << 31) for _ in range(50))]:
            if 0 <= n < 1 << 31:
                assert rules.attention_divide(n, d) == n // d, (n, d)


def test_padded_dims(rules):
    for dim in range(8, 257, 8):
        padded = rules.attention_padded_dim(dim)
        assert padded >= dim and padded in (64, 96, 128, 192, 256)
        assert rules.attention_padded_dim(padded) == padded


def test_workspace_bytes_of_the_library(rules, lib):
    for tokens, batch, heads, kv, dim, positions in (
            (1, 1, 32, 8, 128, 8192), (64, 64, 32, 8, 80, 16384), (512, 1, 8, 8, 200, 9000)):
        body = rules.attention_workspace(tokens, batch, heads, kv, dim, positions, 0)
        assert hip_lib.paged_attention_workspace_bytes(
            tokens, batch, heads, kv, dim, positions) == body + (5 << 20) + 256
    assert hip_lib.paged_attention_workspace_bytes(8192, 1, 32, 8, 128, 8192) == 0
    for bad in ((-1, 1, 8, 8, 64, 64), (1, 0, 8, 8, 64, 64), (1, 1, 9, 8, 64, 1 << 20),
                (1, 1, 8, 0, 64, 64), (1, 1, 8, 8, 264, 1 << 20)):
        assert hip_lib.paged_attention_workspace_bytes(*bad) == 0
    # One partial row a workgroup, 1024 of them at most.
    assert hip_lib.workspace_bytes("qk_norm_rope_bwd", 1000, 128) >= (5 << 20) + 1024 * 128 * 4
