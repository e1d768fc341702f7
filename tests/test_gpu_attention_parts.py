"""Attention over a paged cache where its steps are dealt out in parts, and without:
more sequences than a wave counts at once, every width of the products with every
page size that is copied in a way of its own, many parts of a tile, more sequences
than are counted at all."""
import math

import pytest
import torch

from credit_amd import hip_lib
from tests.test_gpu_paged_attention import BF16, call, check, close, expected, make, workspace

pytestmark = pytest.mark.gpu


def parted(args) -> bool:
    return workspace(args)[1] > 0


# New tokens and positions: a tile a sequence, several small ones, large ones.
SHAPES = {"few": ([1, 1, 2], [700, 90, 1500]), "several": ([60, 1, 130], [1500, 30, 700]),
          "large": ([60, 1, 130], [2300, 30, 2100])}


@pytest.mark.parametrize("page", [16, 8, 12])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("shape", SHAPES.values(), ids=SHAPES)
def test_widths_and_pages(gpu, shape, dim, page):
    args = make(*shape, 2, 1, dim, page, seed=dim + page)
    assert parted(args)
    check(args)
    # The same without parts: the pages of the longest, a few steps.
    short = make([min(n, 90) for n in shape[0]], [min(n, 100) for n in shape[1]], 2, 1, dim, page)
    assert not parted(short)
    check(short)


@pytest.mark.parametrize("page", [64, 8, 5])
@pytest.mark.parametrize("dim", [64, 96, 128, 192])
def test_large_tiles_whole(gpu, dim, page):
    """Of more key heads than small tiles would have a CU each, and few steps; of more
    rows than there are units."""
    args = make([300, 200, 1, 0], [400, 510, 30, 9], 16, 16, dim, page, seed=dim + page)
    assert not parted(args)
    check(args, window=0 if page == 8 else 77)
    args = make([60] * 8, [600] + [100] * 7, 64, 64, dim, page, seed=dim)
    assert not parted(args)
    check(args)


@pytest.mark.parametrize("dim", [8, 72, 80, 104, 136, 200])
@pytest.mark.parametrize("shape", [([2], [900]), ([90], [1300]), ([90], [2200])],
                         ids=["few", "several", "large"])
def test_dims_between_the_widths(gpu, shape, dim):
    args = make(*shape, 3, 1, dim, 16, seed=dim)
    assert parted(args)
    check(args, window=700 if dim % 16 else 0)


@pytest.mark.parametrize("batch", [64, 65, 130, 300])
def test_more_sequences_than_a_wave(gpu, batch):
    """Ragged ones, some without tokens, some without positions."""
    g = torch.Generator().manual_seed(batch)
    kvs = torch.randint(0, 400, (batch,), generator=g).tolist()
    kvs[-1] = 1100
    news = [0 if i % 7 == 3 else 1 for i in range(batch)]
    args = make(news, kvs, 4, 2, 64, 16)
    assert parted(args)
    check(args)
    check(args, window=50)


def test_large_tiles_of_many_sequences(gpu):
    """Sequences beyond the first 64 whose tiles have more than 32 rows."""
    news = [40 if i % 9 == 0 else 1 for i in range(80)]
    args = make([*news, 3000], [n + 30 for n in news] + [3100], 1, 1, 16, 16)
    assert parted(args)
    check(args)


def test_more_sequences_than_are_counted(gpu):
    """A batch without parts, each tile found by a search."""
    batch = 1100
    args = make([i % 3 for i in range(batch)], [i % 40 for i in range(batch)], 2, 1, 16, 16)
    args = (*args[:3], torch.nn.functional.pad(args[3], (0, 40), value=-1), *args[4:])
    assert args[3].shape[1] * 16 > 8 * 32 and not parted(args)
    check(args)


@pytest.mark.parametrize("new", [1, 40])
def test_many_parts_of_a_tile(gpu, new):
    """One key head over a long cache: more parts than a wave joins at once."""
    args = make([new], [70000], 4, 1, 64, 64, loud=1.0)
    assert parted(args)
    check(args)


@pytest.mark.parametrize("window", [1, 33, 64, 65, 1000, 2 ** 31 - 1])
@pytest.mark.parametrize("shape", [([1, 3], [3000, 800]), ([70, 200], [2000, 900]),
                                   ([70, 200], [2400, 900])], ids=["few", "several", "large"])
def test_windows(gpu, shape, window):
    args = make(*shape, 7, 1, 64, 16)
    assert parted(args)
    check(args, window)


@pytest.mark.parametrize("longest", [2000, 2500])  # small tiles, large ones
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_hidden_values_in_parts(gpu, value, longest):
    """Garbage in front of a window, where a step is shared by rows that see it and
    rows that do not."""
    args = make([3, 40], [longest, 1500], 4, 2, 128, 16)
    want = call(args, 100)
    table, page = args[3], 16
    for b, js in ((0, (5, 1000, 1896)), (1, (0, 1359))):
        for j in js:
            for cache in args[1:3]:
                cache[table[b, j // page].long(), j % page] = value
    got = call(args, 100)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graphs_take_turns_with_one_workspace(gpu):
    """Two captured calls of different sequences share one, one behind the other."""
    sets = [make([1], [6000], 8, 1, 128, 16, seed=1), make([1, 1], [900, 5000], 8, 1, 128, 16,
                                                         seed=2)]
    want = [call(a) for a in sets]
    buffer = torch.zeros(max(workspace(a)[1] for a in sets), dtype=torch.uint8, device=gpu)
    outs, graphs = [torch.empty_like(a[0]) for a in sets], []
    for a, out in zip(sets, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            hip_lib.paged_attention(*a, out, cfg=hip_lib.make_cfg(workspace=buffer))
        graphs.append(graph)
    for _ in range(3):
        for out in outs:
            out.zero_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, w[0]) for out, w in zip(outs, want))
        again = [call(a)[0] for a in sets]
        assert all(torch.equal(a, w[0]) for a, w in zip(again, want))


def test_a_padded_batch(gpu):
    """A batch of a fixed size, its last sequences without tokens and positions and
    their rows of pages not filled, as a captured decode step has it."""
    args = list(make([1, 1, 1], [900, 40, 3000], 8, 2, 128, 16))
    want = call(tuple(args))
    spare = 5
    args[0] = torch.cat((args[0], torch.full((spare, 8, 128), math.nan, dtype=BF16, device=gpu)))
    args[3] = torch.cat((args[3], torch.full((spare, args[3].shape[1]), 2 ** 30,
                                             dtype=torch.int32, device=gpu)))
    args[4] = torch.cat((args[4], args[4][-1:].expand(spare)))
    args[5] = torch.cat((args[5], torch.zeros(spare, dtype=torch.int32, device=gpu)))
    out, lse = call(tuple(args))
    (exact, exact_lse), (bound, bound_lse) = expected(
        (args[0][:3], *args[1:3], args[3][:3], args[4][:4], args[5][:3]))
    close(out[:3], exact, bound, "bf16")
    close(lse[:3], exact_lse, bound_lse, "f32")
    assert (out[3:] == 7).all() and (lse[3:] == 7).all()
    assert torch.equal(want[0][1], out[1])  # one part with and without the others
