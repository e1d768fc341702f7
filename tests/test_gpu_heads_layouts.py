"""Paged caches of any order of pages, slots and heads, keys and values in one buffer:
filled and read as those of the usual layout, bit by bit, nothing else touched."""
import itertools

import pytest
import torch

from credit_amd import hip_lib

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
PAGES, KH, DIM = 9, 3, 64


@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("order", itertools.permutations("psh2"), ids="".join)
def test_every_order(gpu, order, page):
    g = torch.Generator().manual_seed(0)
    news, kvs = (30, 1), (70, 40)
    tokens, qh = sum(kvs), 6
    q = torch.randn((sum(news), qh, DIM), generator=g).to(BF16).to(gpu)
    k, v = (torch.randn((tokens, KH, DIM), generator=g).to(BF16).to(gpu) for _ in "kv")
    pages = -(-kvs[0] // page) + -(-kvs[1] // page) + 1
    table = torch.full((2, -(-kvs[0] // page)), -1, dtype=torch.int32)
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    table[0], table[1, :-(-kvs[1] // page)] = perm[:table.shape[1]], perm[
        table.shape[1]:table.shape[1] + -(-kvs[1] // page)]
    slots = torch.cat([table[b, torch.arange(n) // page].long() * page + torch.arange(n) % page
                       for b, n in enumerate(kvs)]).to(gpu)
    table = table.to(gpu)
    start = torch.tensor([0, news[0], sum(news)], dtype=torch.int32, device=gpu)
    lengths = torch.tensor(kvs, dtype=torch.int32, device=gpu)
    pos = torch.arange(tokens, device=gpu)
    freq = hip_lib.rope_frequencies(DIM)[0].to(gpu)

    def run(caches):
        hip_lib.paged_append(k, v, slots, *caches, pos, freq)
        out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=gpu)
        hip_lib.paged_attention(q, *caches, table, start, lengths, out, lse)
        return out, lse

    usual = [torch.full((pages, page, KH, DIM), 3.0, dtype=BF16, device=gpu) for _ in "kv"]
    want = run(usual)
    sizes = {"p": pages, "s": page, "h": KH, "2": 2}
    buffer = torch.full([sizes[c] for c in order] + [DIM + 8], 3.0, dtype=BF16, device=gpu)
    caches = buffer[..., :DIM].permute(*(order.index(c) for c in "2psh"), 4).unbind(0)
    got = run(caches)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(caches, usual))
    assert (buffer[..., DIM:] == 3).all()


def test_tensors_next_to_each_other(gpu):
    """All tensors of the gradients, of norm and rotation and of an attention one behind
    the other in one buffer: none overlaps, none is refused, the values are those of
    tensors of their own."""
    tokens, qh, kh = 7, 6, 2
    g = torch.Generator().manual_seed(1)
    arena, at = torch.zeros(1 << 20, dtype=torch.uint8, device=gpu), 0

    def put(t):
        nonlocal at
        n = t.numel() * t.element_size()
        here = arena[at:at + n].view(t.dtype).view(t.shape)
        at += n
        here.copy_(t)
        return here

    def both(f):
        own = f(lambda t: t.to(gpu))
        for a, b in zip(f(put), own):
            assert torch.equal(a, b)

    xs, dys = ([torch.randn((tokens, h, DIM), generator=g).to(BF16) for h in (qh, kh)]
               for _ in "xy")
    ws = [torch.randn(DIM, generator=g).to(BF16) for _ in "qk"]
    pos, freq = torch.arange(tokens + 1), hip_lib.rope_frequencies(DIM)[0]  # 16-byte units
    rstd = torch.zeros((tokens, qh + kh))

    def training(at):
        q, k, wq, wk, p, f, r, *more = (at(t) for t in (
            *xs, *ws, pos, freq, rstd, *xs, *dys, *xs, *(torch.zeros(DIM) for _ in "qk")))
        p = p[:tokens]
        hip_lib.qk_norm_rope_fwd(q, k, wq, wk, p, f, more[0], more[1], r)
        hip_lib.qk_norm_rope_bwd(q, k, wq, wk, p, f, r, *more[2:])
        return r, *more

    def serving(at):
        q, k_cache, v_cache, table, start, lengths, out, lse = (at(t) for t in (
            xs[0], *(torch.randn((4, 4, kh, DIM), generator=g.manual_seed(2)).to(BF16)
                     for _ in "kv"),
            torch.tensor([[3, 1, 2, 0]], dtype=torch.int32),
            torch.tensor([0, tokens, tokens, tokens], dtype=torch.int32),
            torch.tensor([14, 0, 0, 0], dtype=torch.int32), torch.zeros_like(xs[0]),
            torch.zeros((tokens, qh))))
        hip_lib.paged_attention(q, k_cache, v_cache, table, start[:2], lengths[:1], out, lse)
        return out, lse

    both(training)
    both(serving)
