"""Attention over a paged cache against the oracle, element by element within
counted bounds: lengths, head layouts, pages, windows, hidden values, pages that are
not there, strides, parts, graphs; and the run of norm, rotation, append and
attention that a model's serving step makes."""
import math

import numpy as np
import pytest
import torch

from credit_amd import hip_lib
from oracle import heads as ref
from tests import heads_bounds as bounds

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16

# new tokens, positions, query heads, key heads, dim, page size, window
CASES = [
    ([1], [1], 1, 1, 8, 1, 0),
    ([1], [300], 4, 1, 128, 16, 0),
    ([1], [5000], 8, 1, 128, 16, 0),
    ([1, 1, 1, 1, 1, 1], [1, 2, 31, 32, 33, 65], 8, 2, 64, 16, 0),
    ([1] * 70, [3 * i + 1 for i in range(70)], 4, 4, 64, 32, 0),
    ([1, 3, 0, 2], [0, 1, 50, 200], 2, 1, 96, 3, 0),
    ([4, 2], [700, 130], 8, 1, 128, 64, 0),
    ([70, 1, 130], [300, 65, 130], 14, 2, 80, 24, 0),
    ([40], [40], 4, 4, 256, 32, 0),
    ([40], [1300], 2, 2, 192, 128, 0),
    ([3], [100], 64, 1, 64, 7, 0),
    ([5, 0, 17], [4, 9, 900], 5, 1, 72, 11, 0),
    ([200], [260], 3, 3, 16, 64, 0),
    ([130], [130], 2, 1, 128, 16, 0),
    ([1, 1], [3000, 90], 8, 2, 128, 16, 100),
    ([90, 30], [400, 30], 4, 2, 128, 16, 1),
    ([90, 30], [400, 30], 4, 2, 64, 16, 70),
    ([33, 1, 64], [200, 20, 64], 4, 1, 256, 8, 33),
]


def make(news, kvs, qh, kh, dim, page, seed=0, gpu="cuda", spare=3, loud=2.0):
    """Tensors of a call, every page that no sequence has among the others and full of
    NaN, as are the slots behind a sequence's last position."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in kvs]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(kvs), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    caches = [torch.full((pages, page, kh, dim), math.nan) for _ in "kv"]
    for b, (n, kv) in enumerate(zip(need, kvs)):
        table[b, :n] = order[at:at + n]
        for j in range(n):
            live = min(page, kv - j * page)
            for c in caches:
                c[order[at + j], :live] = torch.randn((live, kh, dim), generator=g)
        at += n
    q_start = torch.tensor([0] + news).cumsum(0).to(torch.int32)
    q = torch.randn((int(q_start[-1]), qh, dim), generator=g) * loud
    k, v = (c.to(BF16).to(gpu) for c in caches)
    return (q.to(BF16).to(gpu), k, v, table.to(gpu), q_start.to(gpu),
            torch.tensor(kvs, dtype=torch.int32).to(gpu))


def np64(t):
    return t.double().cpu().numpy()


def call(args, window=0, scale=None, cfg=None, lse=True):
    q = args[0]
    out = torch.full_like(q, 7.0)
    logs = torch.full(q.shape[:2], 7.0, device=q.device) if lse else None
    hip_lib.paged_attention(*args, out, logs, scale, window, cfg)
    return out, logs


def expected(args, window=0, scale=None):
    q, k, v, table, q_start, kv_len = args
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    host = (np64(q), np64(k), np64(v), table.cpu().numpy(), q_start.tolist(), kv_len.tolist(),
            scale, window)
    return ref.paged_attention(*host), bounds.attention(*host)


def close(got, want, bound, dtype):
    got = np64(got)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    finite = np.isfinite(want)
    assert np.array_equal(got[~finite & ~nan], want[~finite & ~nan])
    got, want, bound = got[finite], want[finite], bound[finite]
    limit = bounds.rounded(bound, want, dtype)
    off = np.abs(got - want)
    assert (off <= limit).all(), (off / limit).max()


def check(args, window=0, scale=None):
    out, lse = call(args, window, scale)
    (want, want_lse), (bound, bound_lse) = expected(args, window, scale)
    close(out, want, bound, "bf16")
    close(lse, want_lse, bound_lse, "f32")
    return out, lse


@pytest.mark.parametrize("case", CASES, ids=str)
def test_attention(gpu, case):
    *shape, window = case
    args = make(*shape)
    out, _ = check(args, window)
    assert torch.equal(call(args, window, lse=False)[0], out)


@pytest.mark.parametrize("scale", [1e-3, 1.0])
def test_scale(gpu, scale):
    check(make([20, 1], [80, 300], 4, 2, 64, 16, loud=1.0), scale=scale)


def test_loud_scores(gpu):
    """Maxima that rise late and by a lot, scores of thousands."""
    args = make([3, 50], [800, 200], 4, 1, 128, 16, loud=60.0)
    check(args, scale=1.0)
    q, k, v, *rest = make([1, 40], [2000, 90], 4, 1, 64, 16, loud=1.0)
    k *= torch.linspace(0, 8, k.shape[0], device=gpu).to(BF16)[:, None, None, None]
    check((q, k, v, *rest))


# ------------------------------------------------ hidden and special values --


def spoil(args, b, j, which, value):
    """Puts a value into position j of sequence b."""
    table, page = args[3], args[1].shape[1]
    args[which][table[b, j // page].long(), j % page] = value


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_hidden_values_change_nothing(gpu, value):
    """Later tokens' keys and values, and those before a window."""
    args = make([60], [150], 4, 2, 64, 16)
    out, lse = call(args, 40)
    for j in (149, 130, 95):
        for which in (1, 2):
            spoil(args, 0, j, which, value)
    got, got_lse = call(args, 40)
    # Token i of position 90 + i sees (50 + i, 90 + i].
    untouched = [i for i in range(60) if not any(50 + i < j <= 90 + i for j in (95, 130, 149))]
    assert len(untouched) >= 5
    assert torch.equal(got[untouched], out[untouched])
    assert torch.equal(got_lse[untouched], lse[untouched])


def test_visible_infinities_and_nan(gpu):
    """Of a value that is seen, whatever its weight, and next to hidden ones."""
    args = make([60], [150], 2, 1, 64, 16, loud=0.5)
    spoil(args, 0, 100, 2, math.inf)
    spoil(args, 0, 120, 2, -math.inf)
    spoil(args, 0, 140, 2, math.nan)
    out, _ = call(args)
    at = torch.arange(60) + 90
    assert out[at < 100].isfinite().all()
    assert (out[(at >= 100) & (at < 120)] == math.inf).all()
    assert out[at >= 120].isnan().all()


def test_scores_of_infinity(gpu):
    """Keys of -inf against positive queries have no weight; a row of nothing else
    is empty; +inf and NaN make their rows NaN."""
    args = make([4], [4], 2, 1, 64, 4)
    args[0].copy_(args[0].abs())
    spoil(args, 0, 0, 1, -math.inf)
    spoil(args, 0, 1, 1, -math.inf)
    spoil(args, 0, 3, 1, math.inf)
    out, lse = check(args)
    assert (out[:2] == 0).all() and (lse[:2] == -math.inf).all()
    assert out[2].isfinite().all() and out[3].isnan().all()


@pytest.mark.parametrize("bad", [-1, 10 ** 6, -2 ** 31])
@pytest.mark.parametrize("shape", [([1, 1], [300, 100]), ([90, 5], [300, 100])], ids=str)
def test_pages_outside_the_cache(gpu, shape, bad):
    args = make(*shape, 4, 1, 128, 16)
    args[3][0, 14] = bad  # positions 224 .. 239 of the first sequence
    check(args)


def test_empty_rows_and_rows_of_no_sequence(gpu):
    """More new tokens than positions; tokens in front of the first sequence and
    behind the last are left."""
    q, k, v, table, q_start, kv_len = make([9, 40], [5, 40], 4, 2, 64, 16)
    q = torch.cat((q[:3], q, q[:5]))
    q_start = q_start + 3
    out, lse = call((q, k, v, table, q_start, kv_len))
    assert (out[:3] == 7).all() and (out[52:] == 7).all() and (lse[52:] == 7).all()
    assert (out[3:7] == 0).all() and (lse[3:7] == -math.inf).all()
    assert (out[7:52] != 7).any(-1).all()


def test_lengths_out_of_range_stay_in_bounds(gpu):
    """A length beyond the row of pages counts as the row's; negative ones are 0."""
    args = make([1, 1, 2], [64, 48, 64], 4, 2, 64, 16)
    want, _ = call(args)
    args[5][0] = 10 ** 9
    args[5][1] = -5
    out, lse = call(args)
    assert torch.equal(out[0], want[0]) and torch.equal(out[2:], want[2:])
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()


def test_no_pages_and_no_tokens(gpu):
    args = list(make([2, 1], [10, 10], 4, 2, 64, 16))
    args[3] = args[3][:, :0]
    out, lse = call(args)
    assert (out == 0).all() and (lse == -math.inf).all()
    args = make([2, 1], [10, 10], 4, 2, 64, 16)
    empty = (args[0][:0], *args[1:4], args[4] * 0, args[5])
    call(empty)
    none = (args[0], *args[1:3], args[3][:0], args[4][:1], args[5][:0])
    out, _ = call(none)
    assert (out == 7).all()


# ------------------------------------------------------------------ layouts --


def test_strides(gpu):
    """Queries as columns of a projection, caches with heads first and in one
    buffer, tables and outputs with room behind their rows."""
    args = make([30, 1], [100, 70], 4, 2, 64, 16)
    want, want_lse = call(args)
    q, k, v, table, *rest = args
    both = torch.stack((k, v), 1).permute(0, 1, 3, 2, 4).contiguous()
    wide = torch.cat((q, q, q), 1)
    room = torch.full((table.shape[0], table.shape[1] + 5), 3, dtype=torch.int32, device=gpu)
    room[:, :table.shape[1]] = table
    out = torch.zeros((q.shape[0], 6, 80), dtype=BF16, device=gpu)
    lse = torch.empty_like(want_lse)
    hip_lib.paged_attention(wide[:, 4:8], both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2),
                            room[:, :table.shape[1]], *rest, out[:, 1:5, 8:72], lse)
    assert torch.equal(out[:, 1:5, 8:72], want) and torch.equal(lse, want_lse)
    out[:, 1:5, 8:72] = 0
    assert not out.any()


def test_far_pages_of_a_large_cache(gpu):
    """Pages whose elements lie behind 2^32 bytes, and behind 2^32 elements."""
    args = make([1, 20], [40, 64], 2, 1, 128, 16)
    want = call(args)
    pages = (5 << 32) // (2 * 16 * 128)
    far = [torch.empty((pages, 16, 1, 128), dtype=BF16, device=gpu) for _ in "kv"]
    table = torch.where(args[3] >= 0, pages - 1 - args[3] * 7, args[3])
    for big, small in zip(far, args[1:3]):
        for i in range(small.shape[0]):
            big[pages - 1 - 7 * i] = small[i]
    got = call((args[0], *far, table, *args[4:]))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------ parts, streams and graphs --


def workspace(args):
    q, k, table = args[0], args[1], args[3]
    n = hip_lib.paged_attention_workspace_bytes(q.shape[0], table.shape[0], q.shape[1], k.shape[2],
                                                q.shape[2], table.shape[1] * k.shape[1])
    return torch.zeros(max(n, 1), dtype=torch.uint8, device=q.device), n


@pytest.mark.parametrize("shape", [([1], [6000], 8, 1), ([1, 1, 1], [6000, 17, 900], 4, 2),
                                   ([60, 1], [4000, 30], 4, 1)], ids=str)
def test_captured_calls_replay(gpu, shape):
    args = make(*shape, 128, 16)
    buffer, n = workspace(args)
    assert n > 0
    out, lse = torch.empty_like(args[0]), torch.empty(args[0].shape[:2], device=gpu)
    plain_out, plain_lse = torch.empty_like(out), torch.empty_like(lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        hip_lib.paged_attention(*args, out, lse, cfg=hip_lib.make_cfg(workspace=buffer))
        hip_lib.paged_attention(*args, plain_out, plain_lse)  # without parts
    for seed in range(3):
        args[0].copy_(make(*shape, 128, 16, seed=seed + 5)[0])
        if seed == 2:
            args[5][0] -= 700  # shorter than when it was captured
        want, want_lse = call(args)
        torch.cuda.synchronize()
        out.zero_(), lse.zero_(), plain_out.zero_(), plain_lse.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        (exact, exact_lse), (bound, bound_lse) = expected(args)
        close(plain_out, exact, bound, "bf16")
        close(plain_lse, exact_lse, bound_lse, "f32")
    assert not buffer[:hip_lib.workspace_bytes("qk_norm_rope_bwd", 1, 1) - 4096].any()


def test_workspace_too_small(gpu):
    args = make([1], [6000], 8, 1, 128, 16)
    _, n = workspace(args)
    small = torch.zeros(n - 256, dtype=torch.uint8, device=gpu)
    with pytest.raises(hip_lib.CreditError, match="workspace"):
        call(args, cfg=hip_lib.make_cfg(workspace=small))


def test_streams_side_by_side(gpu):
    """Calls with parts on two streams at once."""
    sets = [make([1], [6000], 8, 1, 128, 16, seed=s) for s in (1, 2)]
    want = [call(a) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for a, s in zip(sets, streams):
            with torch.cuda.stream(s):
                got.append(call(a))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])


def test_same_bits_from_call_to_call(gpu):
    args = make([1, 1], [9000, 4000], 8, 1, 128, 16)
    first = call(args)
    for _ in range(5):
        again = call(args)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ------------------------------------------------------------- a run of them --


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_serving_run(gpu, layout):
    """Two sequences served in chunks and single tokens, each step norm, rotation and
    append in one launch and attention in another, against attention of all tokens
    at once over keys that the oracle normed and rotated."""
    qh, kh, dim, page, total = 4, 2, 64, 16, (75, 51)
    g = torch.Generator().manual_seed(4)
    qkv = [torch.randn((n, qh + 2 * kh, dim), generator=g).to(BF16).to(gpu) for n in total]
    wq, wk = (1 + 0.2 * torch.randn((2, dim), generator=g)).to(BF16).to(gpu)
    freq, magnitude = hip_lib.rope_frequencies(dim, scaling="yarn", factor=4.0,
                                               original_length=64)
    freq = freq.to(gpu)
    pages = torch.tensor([[7, 2, 0, 9, 4], [1, 3, 5, 6, -1]], dtype=torch.int32, device=gpu)
    caches = [torch.full((10, page, kh, dim), math.nan, dtype=BF16, device=gpu) for _ in "kv"]
    done, outs = [0, 0], [[], []]
    for chunk in ((40, 1), (1, 30), (1, 1), (33, 19)):
        rows = [qkv[b][done[b]:done[b] + n] for b, n in enumerate(chunk)]
        x = torch.cat(rows)
        pos = torch.cat([torch.arange(d, d + n) for d, n in zip(done, chunk)]).to(gpu)
        row = torch.repeat_interleave(torch.arange(2), torch.tensor(chunk)).to(gpu)
        slots = pages[row, pos // page].long() * page + pos % page
        q, k, v = x.split((qh, kh, kh), 1)
        hip_lib.paged_append(k, v, slots, *caches, pos, freq, wk, q, q, wq, layout=layout,
                             magnitude=magnitude)
        done = [d + n for d, n in zip(done, chunk)]
        out = torch.empty((len(x), qh, dim), dtype=BF16, device=gpu)
        start = torch.tensor([0, chunk[0], sum(chunk)], dtype=torch.int32, device=gpu)
        hip_lib.paged_attention(q, *caches, pages, start,
                                torch.tensor(done, dtype=torch.int32, device=gpu), out)
        for b, part in enumerate(out.split(chunk)):
            outs[b].append(part)
    assert done == list(total)
    for b, n in enumerate(total):
        q, k, v = (np64(t) for t in qkv[b].split((qh, kh, kh), 1))
        turned = []
        for t, w in ((q, wq), (k, wk)):
            y, _ = ref.norm_rope(t, np64(w), np.arange(n), np64(freq), layout, magnitude)
            turned.append(np64(torch.from_numpy(y).to(BF16)))  # as the kernels round them
        args = (turned[0], turned[1][None], v[None], [[0]], [0, n], [n], 1 / math.sqrt(dim))
        want, _ = ref.paged_attention(*args)
        bound, _ = bounds.attention(*args)
        # An element that the kernel rounds to the other neighbour is a step off,
        # 2^-7 of it: each score by at most 2^-7 of its terms' size for q and for k.
        size = np.zeros((n, qh))
        for h in range(qh):
            a = np.abs(turned[0][:, h]) @ np.abs(turned[1][:, h // 2]).T
            size[:, h] = (np.tril(a)).max(1)
        flip = np.expm1(2 * 2 * 2.0 ** -7 * size / math.sqrt(dim))
        bound = bound + flip[..., None] * np.abs(v).max()
        close(torch.cat(outs[b]), want, bound, "bf16")
