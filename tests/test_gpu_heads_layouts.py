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
