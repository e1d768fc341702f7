"""Attention over a paged cache on tiles of 128 rows, whole and in parts, where it can
go wrong: maxima that rise late, infinities and NaN that are seen or hidden, pages that
are not there, rows that see nothing, strides, pages beyond 2^32 elements.  Each test
asks the rules whether its call takes such tiles."""
import math

import pytest
import torch

from tests.heads_rules_lib import FEW, MANY, build, way
from tests.test_gpu_paged_attention import BF16, call, check, make, np64, spoil
from credit_amd import hip_lib

pytestmark = pytest.mark.gpu

WHOLE, PARTS = (MANY, False), (MANY, True)
# New tokens, positions, query heads, key heads.
SHAPES = {WHOLE: ([150, 130], [300, 130], 32, 16), PARTS: ([150, 40], [2300, 130], 2, 1)}
both = pytest.mark.parametrize("which", SHAPES, ids=["whole", "parts"])


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    return build(tmp_path_factory.mktemp("rules"))


def ramp(args, b, first, last):
    """Scales the keys of sequence b from `first` to `last` along its positions."""
    q, k, _, table, _, kv_len = args
    kv, page = int(kv_len[b]), k.shape[1]
    at = torch.arange(kv, device=q.device)
    where = table[b, at // page].long(), at % page
    by = torch.linspace(first, last, kv, device=q.device)[:, None, None]
    k[where] = (k[where].float() * by).to(BF16)


def rises(args, b, step, scale):
    """Rows of the last token of sequence b whose scores pass the first step's by more
    than 2^16."""
    q, k, _, table, q_start, kv_len = args
    kv, page = int(kv_len[b]), k.shape[1]
    at = torch.arange(kv, device=q.device)
    keys = k[table[b, at // page].long(), at % page].double()
    token = q[int(q_start[b + 1]) - 1].double()
    keys = keys.repeat_interleave(q.shape[1] // k.shape[2], 1)
    x = (keys * token).sum(-1) * scale  # [positions, heads]
    first = x[:step].amax(0)
    return int(((x.amax(0) - first) * math.log2(math.e) > 16).sum())


@both
@pytest.mark.parametrize("dim", [64, 80, 128, 192])
def test_maxima_that_rise_late(gpu, rules, which, dim):
    args = make(*SHAPES[which], dim, 16, seed=dim)
    ramp(args, 0, 0.0, 16.0)
    assert way(rules, args) == which and rises(args, 0, 64, dim ** -0.5) > 0
    check(args)


@both
@pytest.mark.parametrize("page", [16, 24, 5])
def test_scores_of_thousands(gpu, rules, which, page):
    args = make(*SHAPES[which], 128, page, loud=60.0)
    assert way(rules, args) == which and rises(args, 0, 64, 1.0) > 0
    check(args, scale=1.0)


def test_maxima_that_rise_late_in_wide_heads(gpu, rules):
    """Heads of 256, which small tiles take however many rows there are."""
    args = make([70], [2300], 4, 2, 256, 16)
    ramp(args, 0, 0.0, 16.0)
    assert way(rules, args) == (FEW, True) and rises(args, 0, 32, 1 / 16) > 0
    check(args)


@both
@pytest.mark.parametrize("dim", [64, 80, 128, 192])
@pytest.mark.parametrize("page", [16, 8, 5])
def test_visible_infinities_and_nan(gpu, rules, which, dim, page):
    """Values of the last sequence's new tokens: seen by the tokens behind them, hidden
    from those before."""
    args = make(*SHAPES[which], dim, page, loud=0.5)
    assert way(rules, args) == which
    want, want_lse = call(args)
    new, kv = (shape[0] for shape in SHAPES[which][:2])
    for j, value in ((kv - 90, math.inf), (kv - 70, -math.inf), (kv - 20, math.nan)):
        spoil(args, 0, j, 2, value)
    out, lse = call(args)
    at = torch.arange(new) + kv - new
    one = out[:new]
    assert torch.equal(one[at < kv - 90], want[:new][at < kv - 90])
    assert (one[(at >= kv - 90) & (at < kv - 70)] == math.inf).all()
    assert one[at >= kv - 70].isnan().all()
    assert torch.equal(out[new:], want[new:]) and torch.equal(lse, want_lse)


@both
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_hidden_values_change_nothing(gpu, rules, which, value):
    """Keys and values of later tokens and in front of a window."""
    window = 40 if which == WHOLE else 400  # of 40 positions there would be no parts
    args = make(*SHAPES[which], 64, 16)
    assert way(rules, args, window) == which
    new, kv = (shape[0] for shape in SHAPES[which][:2])
    out, lse = call(args, window)
    spoiled = (0, kv - new - window + 60, kv - 20)
    for j in spoiled:
        for tensor in (1, 2):
            spoil(args, 0, j, tensor, value)
    got, got_lse = call(args, window)
    untouched = [i for i in range(len(out)) if i >= new or not any(
        kv - new + i - window < j <= kv - new + i for j in spoiled)]
    assert len(untouched) > len(out) - 100
    assert torch.equal(got[untouched], out[untouched])
    assert torch.equal(got_lse[untouched], lse[untouched])


@pytest.mark.parametrize("which,shape", [(WHOLE, ([270], [270], 32, 32)),
                                         (PARTS, ([270, 1], [270, 2100], 4, 2))],
                         ids=["whole", "parts"])
def test_scores_of_infinity(gpu, rules, which, shape):
    """Keys of -inf against positive queries have no weight; rows of nothing else are
    empty; +inf makes its rows NaN."""
    args = make(*shape, 64, 16)
    assert way(rules, args) == which
    args[0].copy_(args[0].abs())
    for j in (*range(70), 100, 200):
        spoil(args, 0, j, 1, -math.inf)
    spoil(args, 0, 250, 1, math.inf)
    out, lse = check(args)
    assert (out[:70] == 0).all() and (lse[:70] == -math.inf).all()
    assert out[70:250].isfinite().all() and out[250:270].isnan().all()


@both
@pytest.mark.parametrize("bad", [-1, 10 ** 6, -2 ** 31])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (80, 8), (192, 64), (128, 12)])
def test_pages_outside_the_cache(gpu, rules, which, bad, dim, page):
    args = make(*SHAPES[which], dim, page)
    assert way(rules, args) == which
    new, kv = (shape[0] for shape in SHAPES[which][:2])
    args[3][0, (kv - 100) // page] = bad
    out, _ = check(args)
    seen = (kv - 100) // page * page - (kv - new)  # the first token that sees it
    assert seen > 0 and out[:seen].isfinite().all() and out[seen:new].isnan().all()


@pytest.mark.parametrize("which,shape", [(WHOLE, ([200, 130], [70, 130], 32, 16)),
                                         (PARTS, ([200, 300], [70, 2200], 2, 1))],
                         ids=["whole", "parts"])
def test_empty_rows_and_rows_of_no_sequence(gpu, rules, which, shape):
    """More new tokens than positions, over a whole tile and more; tokens in front of
    the first sequence and behind the last are left."""
    q, k, v, table, q_start, kv_len = make(*shape, 64, 16)
    args = torch.cat((q[:3], q, q[:5])), k, v, table, q_start + 3, kv_len
    assert way(rules, args) == which
    out, lse = call(args)
    end = 3 + sum(shape[0])
    for t in (out, lse):
        assert (t[:3] == 7).all() and (t[end:] == 7).all()
    assert (out[3:133] == 0).all() and (lse[3:133] == -math.inf).all()
    assert (out[133:end] != 7).any(-1).all() and (lse[133:end] != 7).all()
    again, lse_again = check((q, k, v, table, q_start, kv_len))
    assert torch.equal(out[3:end], again) and torch.equal(lse[3:end], lse_again)


@both
def test_strides(gpu, rules, which):
    """Queries as columns of a projection, caches with heads first and in one buffer,
    tables and outputs with room behind their rows."""
    args = make(*SHAPES[which], 64, 16)
    assert way(rules, args) == which
    want, want_lse = call(args)
    q, k, v, table, *rest = args
    heads = q.shape[1]
    both = torch.stack((k, v), 1).permute(0, 1, 3, 2, 4).contiguous()
    wide = torch.cat((q, q, q), 1)
    room = torch.full((table.shape[0], table.shape[1] + 5), 3, dtype=torch.int32, device=gpu)
    room[:, :table.shape[1]] = table
    out = torch.zeros((q.shape[0], heads + 2, 80), dtype=BF16, device=gpu)
    lse = torch.empty_like(want_lse)
    got = out[:, 1:heads + 1, 8:72]
    hip_lib.paged_attention(wide[:, heads:2 * heads], both[:, 0].transpose(1, 2),
                            both[:, 1].transpose(1, 2), room[:, :table.shape[1]], *rest, got, lse)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    got.zero_()
    assert not out.any()


@both
def test_far_pages_of_a_large_cache(gpu, rules, which):
    """Pages whose elements lie behind 2^32 bytes, and behind 2^32 elements."""
    args = make(*SHAPES[which], 128, 16)
    assert way(rules, args) == which
    want = call(args)
    kh = SHAPES[which][3]
    pages = (5 << 32) // (2 * 16 * kh * 128)
    far = [torch.empty((pages, 16, kh, 128), dtype=BF16, device=gpu) for _ in "kv"]
    table = torch.where(args[3] >= 0, pages - 1 - args[3] * 7, args[3])
    for big, small in zip(far, args[1:3]):
        for i in range(small.shape[0]):
            big[pages - 1 - 7 * i] = small[i]
    got = call((args[0], *far, table, *args[4:]))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("columns", [64, 1024, 8192])
@pytest.mark.parametrize("filler", [-1, 2 ** 31 - 1])
def test_tables_wider_than_the_sequences(gpu, columns, filler):
    """A server's table is as wide as its longest context; what lies behind a sequence's
    pages is not looked at."""
    for shape in (([1, 3], [300, 90], 8, 2), ([40, 1], [500, 20], 8, 2),
                  ([300, 20], [420, 30], 4, 1)):
        q, k, v, table, *rest = make(*shape, 64, 16)
        wide = torch.full((2, columns), filler, dtype=torch.int32, device=gpu)
        wide[:, :table.shape[1]] = table
        check((q, k, v, wide, *rest))


@both
def test_same_bits_from_call_to_call(gpu, rules, which):
    args = make(*SHAPES[which], 128, 16)
    assert way(rules, args) == which
    first = call(args)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(call(args), first))
    assert np64(first[0]).any()
