"""Where paged caches may lie: any strides but the last, keys and values in one buffer,
as long as no element is shared (credit_amd/csrc/heads_rules.hpp).  No GPU."""
import ctypes
import itertools
import random
import shutil
import subprocess
from pathlib import Path

import pytest

from credit_amd import hip_lib
from tests.test_heads_refusals import CONFIG, SHAPE, CreditPages, call, heads, pages

PLACE = ctypes.c_int64 * 8


@pytest.fixture(scope="module")
def places(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    source = Path(__file__).resolve().parent / "cpp" / "heads_places_query.cpp"
    out = tmp_path_factory.mktemp("places") / "heads_places.so"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", str(source), "-o",
                    str(out)], check=True)
    lib = ctypes.CDLL(str(out))
    lib.places_apart.argtypes, lib.places_apart_within.argtypes = [PLACE, PLACE], [PLACE]
    return lib


def vectors(p):
    at, run, step, outer, count, width, lead, leads = p
    return [range(at + i * lead + j * run + k * step, at + i * lead + j * run + k * step + width)
            for i in range(leads) for j in range(outer) for k in range(count)]


def test_apart_share_no_byte(places):
    """What is called apart is, over places small enough to count."""
    rng = random.Random(0)
    found = within = 0
    for _ in range(20000):
        ps = [(1000 + rng.randrange(60), rng.choice((0, 3, 4, 8, 12, 16, 24, 31)),
               rng.choice((0, 2, 3, 4, 6, 8)), rng.randrange(1, 4), rng.randrange(1, 4),
               rng.randrange(1, 6), rng.choice((0, 4, 8, 16, 24, 48, 50)), rng.randrange(1, 4))
              for _ in "ab"]
        if rng.random() < 0.7:
            ps[1] = (ps[1][0], *ps[0][1:3], *ps[1][3:6], ps[0][6], ps[1][7])
        a, b = (PLACE(*p) for p in ps)
        bytes_a, bytes_b = (set(itertools.chain(*vectors(p))) for p in ps)
        if places.places_apart(a, b):
            found += 1
            assert not bytes_a & bytes_b, ps
        if places.places_apart_within(a):
            within += 1
            assert len(bytes_a) == sum(map(len, vectors(ps[0]))), ps[0]
        assert places.places_apart(a, b) == places.places_apart(b, a)
    assert found > 1000 and within > 1000


# Orders of (pages, slots, heads), with the place of keys and values (2) among them, from
# the outermost to the innermost; the elements of a head come last.
ORDERS = [o for o in itertools.permutations("psh2")]


def caches(order, sizes, width):
    """(strides of p, s, h and the distance of the values) in units of `width`'s unit."""
    stride, at = {}, width
    for level in reversed(order):
        stride[level] = at
        at *= sizes[level]
    return stride


@pytest.mark.parametrize("order", ORDERS, ids="".join)
def test_every_order_of_one_buffer(places, order):
    for sizes in ({"p": 5, "s": 16, "h": 3, "2": 2}, {"p": 1, "s": 1, "h": 8, "2": 2},
                  {"p": 4, "s": 1, "h": 1, "2": 2}, {"p": 3, "s": 7, "h": 1, "2": 2}):
        st = caches(order, sizes, 64)
        k, v = (PLACE(4096 + i * st["2"], st["s"], st["h"], sizes["s"], sizes["h"], 64, st["p"],
                      sizes["p"]) for i in range(2))
        assert places.places_apart_within(k) and places.places_apart_within(v)
        assert places.places_apart(k, v) and places.places_apart(v, k)
        near = PLACE(4096 + st["2"] - 2, *v[1:])  # an element too early
        assert not places.places_apart(k, near)


@pytest.mark.parametrize("order", ORDERS, ids="".join)
def test_the_library_takes_every_order(lib, order):
    """The calls below are refused for their other tensors alone."""
    st = caches(order, {"p": 100, "s": 16, "h": 8, "2": 2}, 64)
    k, v, near = (CreditPages((8 << 32) + at, st["p"], st["s"], st["h"], 100, 16, 8)
                  for at in (0, 2 * st["2"], 2 * st["2"] - 16))
    for op, name in (("paged_append", "q"), ("paged_attention", "out")):
        assert call(lib, op, "bf16", k_cache=k, v_cache=v, **{name: heads(8 << 32)}) == CONFIG
        assert hip_lib.last_error() in ("k_cache overlaps q", "out overlaps k_cache")
    assert call(lib, "paged_append", "bf16", k_cache=k, v_cache=near) == CONFIG
    assert hip_lib.last_error() == "k_cache overlaps v_cache"


def test_caches_that_overlap_themselves(lib):
    for op in ("paged_append", "paged_attention"):
        for bad in (dict(page=8000), dict(slot=500), dict(head=60), dict(page=512, slot=512),
                    dict(page=64, slot=512 * 99, head=64), dict(page=0)):
            assert call(lib, op, "bf16", k_cache=pages(3 << 32, **bad)) == SHAPE, bad
            assert "overlap" in hip_lib.last_error()
