"""The operators on heads at the limits of their kernels' variants: calls beyond the
last-level cache, which take nontemporal accesses, norms of numbers near the ends of
fp32, gradients on two streams at once."""
import numpy as np
import pytest
import torch

from credit_amd import hip_lib
from tests.heads_bounds import E

pytestmark = pytest.mark.gpu

LARGE = 30000, 20, 4, 128  # tokens, query heads, key heads, dim: 351 MiB in and out


@pytest.fixture(scope="module")
def large():
    g = torch.Generator(device="cuda").manual_seed(0)
    tokens, qh, kh, dim = LARGE
    randn = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()
    xs, dys = ([randn(tokens, h, dim) for h in (qh, kh)] for _ in "xy")
    ws = [1 + randn(dim) / 8 for _ in "qk"]
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda")
    return xs, ws, dys, pos, hip_lib.rope_frequencies(dim)[0].cuda()


def pieces(n, each=5000):
    return [slice(i, min(i + each, n)) for i in range(0, n, each)]


def test_large_forwards_match_small_ones(gpu, large):
    """Bit by bit: an element's arithmetic does not depend on the variant."""
    xs, ws, _, pos, freq = large
    outs, again = ([torch.empty_like(x) for x in xs] for _ in range(2))
    rstd, rstd_again = (torch.empty(LARGE[0], sum(LARGE[1:3]), device=gpu) for _ in range(2))
    hip_lib.qk_norm_rope_fwd(*xs, *ws, pos, freq, *outs, rstd)
    for p in pieces(LARGE[0]):
        hip_lib.qk_norm_rope_fwd(*(x[p] for x in xs), *ws, pos[p], freq, *(y[p] for y in again),
                                 rstd_again[p])
    assert all(torch.equal(a, b) for a, b in zip((*outs, rstd), (*again, rstd_again)))
    hip_lib.rope(xs[0], pos, freq, outs[0], xs[1], outs[1])
    for p in pieces(LARGE[0]):
        hip_lib.rope(xs[0][p], pos[p], freq, again[0][p], xs[1][p], again[1][p])
    assert all(torch.equal(a, b) for a, b in zip(outs, again))


def test_large_appends_match_small_ones(gpu, large):
    (q, k), (wq, wk), (_, v), pos, freq = large
    tokens, _, kh, dim = LARGE
    page = 16
    pages = -(-tokens // page) + 3
    slots = torch.randperm(pages * page, device=gpu)[:tokens]
    slots[::100] = -1
    got, want = ([torch.full((pages, page, kh, dim), 3.0, dtype=torch.bfloat16, device=gpu)
                  for _ in "kv"] for _ in range(2))
    out, again = torch.empty_like(q), torch.empty_like(q)
    hip_lib.paged_append(k, v, slots, *got, pos, freq, wk, q, out, wq)
    for p in pieces(tokens):
        hip_lib.paged_append(k[p], v[p], slots[p], *want, pos[p], freq, wk, q[p], again[p], wq)
    assert torch.equal(out, again) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_large_gradients_match_small_ones(gpu, large):
    """dq and dk bit by bit.  dweight against the sum in 64 bits: a term dy x rstd has
    two roundings; a group of lanes adds at most ceil(units / groups) RUN of them, the
    workgroup its 32 groups', the last kernel 32 runs of rows, and the longest chain of
    these is below 256."""
    xs, ws, dys, pos, freq = large
    rstd = torch.empty(LARGE[0], sum(LARGE[1:3]), device=gpu)
    hip_lib.qk_norm_rope_fwd(*xs, *ws, pos, freq, *(torch.empty_like(x) for x in xs), rstd)
    dxs, again = ([torch.empty_like(x) for x in xs] for _ in range(2))
    dws, spare = ([torch.empty(128, device=gpu) for _ in xs] for _ in range(2))
    hip_lib.qk_norm_rope_bwd(*xs, *ws, pos, freq, rstd, *dys, *dxs, *dws)
    for p in pieces(LARGE[0]):
        hip_lib.qk_norm_rope_bwd(*(x[p] for x in xs), *ws, pos[p], freq, rstd[p],
                                 *(d[p] for d in dys), *(d[p] for d in again), *spare)
    assert all(torch.equal(a, b) for a, b in zip(dxs, again))
    hip_lib.qk_norm_rope_bwd(*xs, *ws, None, None, rstd, *dys, *dxs, *dws)
    at = 0
    for x, dy, dw in zip(xs, dys, dws):
        want, size = (torch.zeros(128, dtype=torch.float64, device=gpu) for _ in range(2))
        for p in pieces(LARGE[0]):
            terms = dy[p].double() * x[p].double() * rstd[p, at:at + x.shape[1], None].double()
            want += terms.sum((0, 1))
            size += terms.abs().sum((0, 1))
        at += x.shape[1]
        assert ((dw.double() - want).abs() <= (256 + 2) * E * size).all()


@pytest.mark.parametrize("eps", [0.0, 1e-40, 1e-30])
@pytest.mark.parametrize("size", [1e-22, 1e-18, 1e-12, 1.0, 1e12, 1e17])
def test_norms_near_the_ends_of_fp32(gpu, size, eps):
    """rstd within its bound where the mean is a normal number, or nothing beside eps:
    a subnormal eps is itself off by at most 2^-149."""
    dim = 64
    rng = np.random.default_rng(0)
    host = (size * rng.choice([-1.0, 1.0], (3, 2, dim))).astype(np.float32)
    x = torch.from_numpy(host).to(gpu)
    one = torch.ones(dim, device=gpu)
    rstd, outs = torch.empty((3, 4), device=gpu), [torch.empty_like(x) for _ in "qk"]
    hip_lib.qk_norm_rope_fwd(x, x.clone(), one, one, None, None, *outs, rstd, eps)
    mean = np.mean(host.astype(np.float64) ** 2, -1) + float(np.float32(eps))
    got = rstd[:, :2].double().cpu().numpy()
    assert np.isfinite(got).all()
    if size > 1e-19 or eps > 1e-35:
        want = mean ** -0.5
        # 22 roundings of the sum, the mean's two, halved; the root's two.
        assert (np.abs(got - want) <= ((22 + 2) / 2 + 2) * E * want).all()
    # Elements of one size norm to 1 where eps is nothing beside their mean, with the
    # bound above for rstd, and a rounding of each product.
    if size > 1e-19 and eps <= 1e-8 * size * size:
        assert (np.abs(outs[0].abs().cpu().numpy() - 1) <= (14 + 2) * E + 1e-8).all()


def test_gradients_on_two_streams(gpu):
    g = torch.Generator().manual_seed(3)
    sets = []
    for tokens in (3000, 1111):
        xs, dys = ([torch.randn((tokens, h, 64), generator=g).to(gpu) for h in (4, 2)]
                   for _ in "xy")
        ws = [torch.randn(64, generator=g).to(gpu) for _ in "qk"]
        pos, freq = torch.arange(tokens, device=gpu), hip_lib.rope_frequencies(64)[0].to(gpu)
        rstd = torch.rand((tokens, 6), generator=g).to(gpu)
        sets.append((xs, ws, pos, freq, rstd, dys))

    def run(s):
        xs, ws, pos, freq, rstd, dys = s
        out = [torch.empty_like(t) for t in (*xs, *ws)]
        hip_lib.qk_norm_rope_bwd(*xs, *ws, pos, freq, rstd, *dys, *out)
        return out

    want = [run(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        got = []
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(run(s))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
