"""Rotary positions, normed rotation with its gradients and the append to a paged
cache against the oracle, element by element within counted bounds."""
import numpy as np
import pytest
import torch

from credit_amd import hip_lib
from oracle import heads as ref
from tests import heads_bounds as bounds
from tests.heads_bounds import DTYPES

pytestmark = pytest.mark.gpu

# tokens, query heads, key heads, dim, rot: every unit and group size, odd ones too.
SHAPES = [(1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (3, 5, 1, 7, 4), (5, 8, 2, 64, 32),
          (2, 14, 2, 80, 40), (33, 3, 3, 96, 96), (7, 2, 1, 256, 128), (4, 3, 2, 512, 512),
          (9, 4, 4, 33, 0), (130, 1, 1, 130, 100), (300, 7, 1, 72, 64), (2, 2, 2, 511, 510)]


def make(tokens, heads, dim, dtype, seed, gpu):
    g = torch.Generator().manual_seed(seed)
    scale = torch.rand((heads, 1), generator=g) * 3 + 0.1
    return (torch.randn((tokens, heads, dim), generator=g) * scale).to(DTYPES[dtype]).to(gpu)


def rotation(tokens, rot, seed, gpu, far=0):
    g = torch.Generator().manual_seed(seed)
    pos = torch.randint(-5, 5000, (tokens,), generator=g) + far
    freq = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) / max(1, rot // 2))
    return pos.to(gpu), freq.float().to(gpu)


def np64(t):
    return t.double().cpu().numpy()


def close(got, want, bound):
    off = np.abs(np64(got) - want)
    assert np.isfinite(np64(got)).all()
    assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rope_and_its_gradient(gpu, shape, dtype, layout):
    tokens, qh, kh, dim, rot = shape
    q, k = make(tokens, qh, dim, dtype, 1, gpu), make(tokens, kh, dim, dtype, 2, gpu)
    pos, freq = rotation(tokens, rot, 3, gpu)
    for transposed in (False, True):
        outs = torch.empty_like(q), torch.empty_like(k)
        hip_lib.rope(q, pos, freq, outs[0], k, outs[1], layout, 1.25, transposed)
        for x, y in zip((q, k), outs):
            args = (np64(x), np64(pos), np64(freq), layout, 1.25, transposed)
            want = ref.rope(*args)
            bound = bounds.rotated(np64(x), 0.0, np64(pos), np64(freq), layout, 1.25)
            close(y, want, bounds.rounded(bound, want, dtype))
            assert torch.equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("far", [10 ** 6, 2 ** 31 - 10000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_far_positions(gpu, dtype, far):
    q = make(64, 3, 128, dtype, 5, gpu)
    pos, freq = rotation(64, 128, 6, gpu, far)
    out = torch.empty_like(q)
    hip_lib.rope(q, pos, freq, out)
    want = ref.rope(np64(q), np64(pos), np64(freq))
    bound = bounds.rotated(np64(q), 0.0, np64(pos), np64(freq), "half", 1.0)
    close(out, want, bounds.rounded(bound, want, dtype))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_norm_rope(gpu, shape, dtype, layout):
    tokens, qh, kh, dim, rot = shape
    xs = make(tokens, qh, dim, dtype, 1, gpu), make(tokens, kh, dim, dtype, 2, gpu)
    ws = [make(1, 1, dim, dtype, s, gpu).view(dim) for s in (3, 4)]
    pos, freq = rotation(tokens, rot, 5, gpu)
    outs = [torch.empty_like(x) for x in xs]
    rstd = torch.empty((tokens, qh + kh), device=gpu)
    hip_lib.qk_norm_rope_fwd(*xs, *ws, pos, freq, *outs, rstd, 1e-5, layout, 0.75)
    for x, w, y, r in zip(xs, ws, outs, (rstd[:, :qh], rstd[:, qh:])):
        want, wr = ref.norm_rope(np64(x), np64(w), np64(pos), np64(freq), layout, 0.75, 1e-5)
        bound = bounds.norm_rope(np64(x), np64(w), np64(pos), np64(freq), layout, 0.75, 1e-5)
        close(y, want, bounds.rounded(bound, want, dtype))
        close(r, wr, wr * bounds.rstd_error(dim))
    dys = make(tokens, qh, dim, dtype, 7, gpu), make(tokens, kh, dim, dtype, 8, gpu)
    dxs = [torch.empty_like(x) for x in xs]
    dws = [torch.empty(dim, device=gpu) for _ in range(2)]
    hip_lib.qk_norm_rope_bwd(*xs, *ws, pos, freq, rstd, *dys, *dxs, *dws, layout, 0.75)
    for x, w, r, dy, dx, dw in zip(xs, ws, (rstd[:, :qh], rstd[:, qh:]), dys, dxs, dws):
        args = (np64(x), np64(w), np64(r), np64(dy), np64(pos), np64(freq), layout, 0.75)
        want, want_w = ref.norm_rope_bwd(*args)
        bound, bound_w = bounds.norm_rope_bwd(*args)
        close(dx, want, bounds.rounded(bound, want, dtype))
        close(dw, want_w, bound_w + 1e-38)


@pytest.mark.parametrize("tokens", [2000, 20000])
def test_many_tokens_share_workgroups(gpu, tokens):
    """More units than a launch has groups, heads that a group takes in turn."""
    xs = make(tokens, 6, 64, "bf16", 1, gpu), make(tokens, 1, 64, "bf16", 2, gpu)
    ws = [make(1, 1, 64, "bf16", s, gpu).view(64) for s in (3, 4)]
    dys = make(tokens, 6, 64, "bf16", 5, gpu), make(tokens, 1, 64, "bf16", 6, gpu)
    pos, freq = rotation(tokens, 64, 7, gpu)
    outs, dxs = ([torch.empty_like(x) for x in xs] for _ in range(2))
    rstd, dws = torch.empty((tokens, 7), device=gpu), [torch.empty(64, device=gpu) for _ in "qk"]
    hip_lib.qk_norm_rope_fwd(*xs, *ws, pos, freq, *outs, rstd)
    hip_lib.qk_norm_rope_bwd(*xs, *ws, pos, freq, rstd, *dys, *dxs, *dws)
    for x, w, y, r, dy, dx, dw in zip(xs, ws, outs, (rstd[:, :6], rstd[:, 6:]), dys, dxs, dws):
        at = np64(pos), np64(freq)
        want, _ = ref.norm_rope(np64(x), np64(w), *at)
        close(y, want, bounds.rounded(bounds.norm_rope(np64(x), np64(w), *at, "half", 1.0, 1e-6),
                                      want, "bf16"))
        args = (np64(x), np64(w), np64(r), np64(dy), *at)
        want, want_w = ref.norm_rope_bwd(*args)
        bound, bound_w = bounds.norm_rope_bwd(*args, "half", 1.0)
        close(dx, want, bounds.rounded(bound, want, "bf16"))
        close(dw, want_w, bound_w)
    again = [torch.empty(64, device=gpu) for _ in "qk"]
    hip_lib.qk_norm_rope_bwd(*xs, *ws, pos, freq, rstd, *dys, *dxs, *again)
    assert all(torch.equal(a, b) for a, b in zip(dws, again))


def test_gradient_against_differences(gpu):
    """fp32, along random directions: the loss changes by the gradient, up to the
    forward's own roundings (an output's bound a step's length) and the third
    derivative's part, 1e-4 of the change at steps of 1e-2 of the inputs."""
    tokens, dim = 6, 48
    xs = make(tokens, 3, dim, "f32", 1, gpu), make(tokens, 2, dim, "f32", 2, gpu)
    ws = [make(1, 1, dim, "f32", s, gpu).view(dim) for s in (3, 4)]
    pos, freq = rotation(tokens, 32, 5, gpu)
    dys = make(tokens, 3, dim, "f32", 6, gpu), make(tokens, 2, dim, "f32", 7, gpu)

    def forward(xs, ws):
        outs = [torch.empty_like(x) for x in xs]
        rstd = torch.empty((tokens, 5), device=gpu)
        hip_lib.qk_norm_rope_fwd(*xs, *ws, pos, freq, *outs, rstd)
        return sum((np64(o) * np64(dy)).sum() for o, dy in zip(outs, dys)), rstd

    _, rstd = forward(xs, ws)
    dxs, dws = [torch.empty_like(x) for x in xs], [torch.empty(dim, device=gpu) for _ in ws]
    hip_lib.qk_norm_rope_bwd(*xs, *ws, pos, freq, rstd, *dys, *dxs, *dws)
    noise = sum((np.abs(np64(dy)) * bounds.norm_rope(np64(x), np64(w), np64(pos), np64(freq),
                                                     "half", 1.0, 1e-6)).sum()
                for x, w, dy in zip(xs, ws, dys))
    h = 1e-2
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        vx = [torch.randn(x.shape, generator=g).to(gpu) * x.abs().mean() for x in xs]
        vw = [torch.randn(w.shape, generator=g).to(gpu) for w in ws]
        plus = [x + h * v for x, v in zip(xs, vx)], [w + h * v for w, v in zip(ws, vw)]
        minus = [x - h * v for x, v in zip(xs, vx)], [w - h * v for w, v in zip(ws, vw)]
        change = (forward(*plus)[0] - forward(*minus)[0]) / (2 * h)
        terms = [np64(d) * np64(v) for d, v in zip(dxs + dws, vx + vw)]
        want = sum(t.sum() for t in terms)
        size = sum(np.abs(t).sum() for t in terms)
        assert abs(change - want) <= noise / h + 1e-3 * size


# ------------------------------------------------------------------ layouts --


def test_columns_of_one_projection_in_place(gpu):
    """Queries and keys as column ranges of one buffer, normed where they lie; the
    values between and behind them stay."""
    tokens, qh, kh, dim = 37, 6, 2, 64
    qkv = make(tokens, qh + 2 * kh, dim, "bf16", 1, gpu)
    want = [torch.empty((tokens, n, dim), dtype=qkv.dtype, device=gpu) for n in (qh, kh)]
    ws = [make(1, 1, dim, "bf16", s, gpu).view(dim) for s in (2, 3)]
    pos, freq = rotation(tokens, dim, 4, gpu)
    parts = qkv.split((qh, kh, kh), 1)
    hip_lib.qk_norm_rope_fwd(parts[0], parts[1], *ws, pos, freq, *want)
    v = parts[2].clone()
    hip_lib.qk_norm_rope_fwd(parts[0], parts[1], *ws, pos, freq, parts[0], parts[1])
    assert torch.equal(parts[0], want[0]) and torch.equal(parts[1], want[1])
    assert torch.equal(parts[2], v)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_offsets(gpu, dtype):
    """Heads outside tokens, odd distances and odd first elements, broadcast inputs."""
    tokens, heads, dim = 11, 3, 64
    x = make(tokens, heads, dim, dtype, 1, gpu)
    pos, freq = rotation(tokens, dim, 2, gpu)
    want = torch.empty_like(x)
    hip_lib.rope(x, pos, freq, want)
    outer = x.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros((tokens, heads, dim + 3), dtype=x.dtype, device=gpu)
    wide[..., 1:dim + 1] = x
    for src in (outer, wide[..., 1:dim + 1]):
        out = torch.full((heads, tokens, dim + 5), 9.0, dtype=x.dtype, device=gpu)
        hip_lib.rope(src, pos, freq, out.transpose(0, 1)[..., 3:dim + 3])
        assert torch.equal(out.transpose(0, 1)[..., 3:dim + 3], want)
        assert (out[..., :3] == 9).all() and (out[..., dim + 3:] == 9).all()
    same = x[:1, :1].expand(tokens, heads, dim)
    out = torch.empty_like(x)
    hip_lib.rope(same, pos, freq, out)
    hip_lib.rope(same.contiguous(), pos, freq, want)
    assert torch.equal(out, want)


def test_gradients_in_place(gpu):
    tokens, dim = 50, 128
    xs = make(tokens, 4, dim, "bf16", 1, gpu), make(tokens, 2, dim, "bf16", 2, gpu)
    dys = make(tokens, 4, dim, "bf16", 3, gpu), make(tokens, 2, dim, "bf16", 4, gpu)
    ws = [make(1, 1, dim, "bf16", s, gpu).view(dim) for s in (5, 6)]
    pos, freq = rotation(tokens, dim, 7, gpu)
    rstd = torch.empty((tokens, 6), device=gpu)
    hip_lib.qk_norm_rope_fwd(*xs, *ws, pos, freq, *(torch.empty_like(x) for x in xs), rstd)
    want, dws = [torch.empty_like(x) for x in xs], [torch.empty(dim, device=gpu) for _ in ws]
    hip_lib.qk_norm_rope_bwd(*xs, *ws, pos, freq, rstd, *dys, *want, *dws)
    for which in range(2):
        ins, outs = [x.clone() for x in xs], [d.clone() for d in dys]
        target = outs if which == 0 else ins
        again = [torch.empty(dim, device=gpu) for _ in ws]
        hip_lib.qk_norm_rope_bwd(*ins, *ws, pos, freq, rstd, *outs, *target, *again)
        assert all(torch.equal(a, b) for a, b in zip(target, want))
        assert all(torch.equal(a, b) for a, b in zip(again, dws))


def test_unturned_elements_keep_to_themselves(gpu):
    """NaN and infinities behind the rotated part reach no other element."""
    for layout in ("half", "interleaved"):
        for dim, rot in ((64, 32), (33, 8), (72, 64)):
            x = make(4, 2, dim, "bf16", 1, gpu)
            pos, freq = rotation(4, rot, 2, gpu)
            want = torch.empty_like(x)
            hip_lib.rope(x, pos, freq, want, layout=layout)
            x[..., rot + 1] = float("nan")
            x[..., rot] = float("inf")
            out = torch.empty_like(x)
            hip_lib.rope(x, pos, freq, out, layout=layout)
            assert torch.equal(out[..., :rot], want[..., :rot])
            assert torch.equal(out[..., rot + 2:], want[..., rot + 2:])
            assert out[..., rot].isinf().all() and out[..., rot + 1].isnan().all()


def test_zero_heads_norm_to_zero(gpu):
    x = make(3, 2, 64, "f32", 1, gpu)
    x[1] = 0.0
    w = torch.ones(64, device=gpu)
    pos, freq = rotation(3, 64, 2, gpu)
    out, rstd = torch.empty_like(x), torch.empty((3, 4), device=gpu)
    hip_lib.qk_norm_rope_fwd(x, x, w, w, pos, freq, out, torch.empty_like(x), rstd, 1e-6)
    assert (out[1] == 0).all()
    np.testing.assert_allclose(np64(rstd[1]), 1e3, rtol=1e-6)


# ------------------------------------------------------------------- append --


@pytest.mark.parametrize("queries", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("shape", [(1, 4, 1, 64, 64, 16), (40, 6, 3, 128, 64, 7),
                                   (9, 2, 2, 33, 20, 1), (300, 8, 8, 80, 0, 24)], ids=str)
def test_append(gpu, shape, norm, queries):
    tokens, qh, kh, dim, rot, page = shape
    g = torch.Generator().manual_seed(9)
    pages = -(-tokens // page) + 5
    q, k, v = (make(tokens, n, dim, "bf16", s, gpu) for n, s in ((qh, 1), (kh, 2), (kh, 3)))
    ws = [make(1, 1, dim, "bf16", s, gpu).view(dim) for s in (4, 5)]
    pos, freq = rotation(tokens, rot, 6, gpu)
    caches = [torch.randn((pages, page, kh, dim), generator=g).bfloat16().to(gpu) for _ in "kv"]
    before = [np64(c) for c in caches]
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    slots[tokens // 2:tokens // 2 + tokens // 8] = -1
    if tokens > 20:
        slots[3], slots[5] = pages * page, 2 ** 62
    q_out = torch.empty_like(q)
    more = dict(q=q, q_out=q_out, q_weight=ws[0] if norm else None) if queries else {}
    hip_lib.paged_append(k, v, slots.to(gpu), *caches, pos if rot else None, freq if rot else None,
                         ws[1] if norm else None, magnitude=1.5, **more)
    at = np64(pos), np64(freq)
    for x, w, got in ((k, ws[1], caches[0]), (q, ws[0], q_out if queries else None)):
        if got is None:
            continue
        if norm:
            new, _ = ref.norm_rope(np64(x), np64(w), *at, "half", 1.5)
            bound = bounds.norm_rope(np64(x), np64(w), *at, "half", 1.5, 1e-6)
        else:
            new = ref.rope(np64(x), *at, "half", 1.5)
            bound = bounds.rotated(np64(x), 0.0, *at, "half", 1.5)
        bound = bounds.rounded(bound, new, "bf16")
        if x is k:
            new = ref.append(before[0], new, slots.tolist())
            bound = ref.append(np.zeros(new.shape), bound, slots.tolist())
        close(got, new, bound)
    want_v = ref.append(before[1], np64(v), slots.tolist())
    assert np.array_equal(np64(caches[1]), want_v)


def test_append_to_caches_of_one_buffer_heads_first(gpu):
    """Keys and values in one [pages, 2, heads, page, dim] buffer."""
    tokens, kh, dim, page, pages = 21, 3, 64, 8, 5
    k, v = (make(tokens, kh, dim, "bf16", s, gpu) for s in (1, 2))
    both = torch.zeros((pages, 2, kh, page, dim), dtype=torch.bfloat16, device=gpu)
    caches = [both[:, i].transpose(1, 2) for i in range(2)]
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(3))[:tokens]
    hip_lib.paged_append(k, v, slots.to(gpu), *caches)
    for cache, new in zip(caches, (k, v)):
        want = ref.append(np.zeros(cache.shape), np64(new), slots.tolist())
        assert np.array_equal(np64(cache), want)


def test_append_far_into_a_large_cache(gpu):
    """Slots whose elements lie behind 2^32 bytes."""
    pages, page, dim = 70000, 256, 128
    cache = torch.zeros((pages, page, 1, dim), dtype=torch.bfloat16, device=gpu)
    small = torch.zeros((pages, page, 1, dim), dtype=torch.bfloat16, device=gpu)
    k = make(3, 1, dim, "bf16", 1, gpu)
    slots = torch.tensor([pages * page - 1, 0, (1 << 32) // (2 * dim) + 5], device=gpu)
    hip_lib.paged_append(k, k, slots, cache, small)
    for c in (cache, small):
        assert torch.equal(c.view(-1, 1, dim)[slots], k)
        c.view(-1, 1, dim)[slots] = 0
        assert not c.view(torch.int64).any()


# ------------------------------------------------------- streams and graphs --


def test_captured_calls_replay(gpu):
    tokens, dim = 40, 128
    xs = make(tokens, 8, dim, "bf16", 1, gpu), make(tokens, 2, dim, "bf16", 2, gpu)
    dys = make(tokens, 8, dim, "bf16", 3, gpu), make(tokens, 2, dim, "bf16", 4, gpu)
    ws = [make(1, 1, dim, "bf16", s, gpu).view(dim) for s in (5, 6)]
    pos, freq = rotation(tokens, dim, 7, gpu)
    rstd = torch.empty((tokens, 10), device=gpu)
    outs, dxs = ([torch.empty_like(x) for x in xs] for _ in range(2))
    dws = [torch.empty(dim, device=gpu) for _ in ws]
    caches = [torch.zeros((8, 16, 2, dim), dtype=torch.bfloat16, device=gpu) for _ in "kv"]
    slots = torch.arange(tokens, device=gpu) * 3
    n = hip_lib.workspace_bytes("qk_norm_rope_bwd", tokens, dim)
    ws_buffer = torch.zeros(n, dtype=torch.uint8, device=gpu)

    def step(cfg=None):
        hip_lib.qk_norm_rope_fwd(*xs, *ws, pos, freq, *outs, rstd, cfg=cfg)
        hip_lib.qk_norm_rope_bwd(*xs, *ws, pos, freq, rstd, *dys, *dxs, *dws, cfg=cfg)
        hip_lib.paged_append(outs[1], xs[1], slots, *caches, cfg=cfg)

    results = [rstd, *outs, *dxs, *dws, *caches]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(hip_lib.CreditError, match="workspace"):
            hip_lib.qk_norm_rope_bwd(*xs, *ws, pos, freq, rstd, *dys, *dxs, *dws)
        step(hip_lib.make_cfg(workspace=ws_buffer))
    for seed in range(3):
        for t in (*xs, *dys):
            t.copy_(make(*t.shape, "bf16", 20 + seed, gpu))
        slots += 1
        for c in caches:
            c.zero_()
        step()
        torch.cuda.synchronize()
        want = [t.clone() for t in results]
        for t in results:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(results, want))


def test_another_stream(gpu):
    xs = make(4000, 8, 128, "bf16", 1, gpu), make(4000, 8, 128, "bf16", 2, gpu)
    pos, freq = rotation(4000, 128, 3, gpu)
    want, got = ([torch.empty_like(x) for x in xs] for _ in range(2))
    hip_lib.rope(xs[0], pos, freq, want[0], xs[1], want[1])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        hip_lib.rope(xs[0], pos, freq, got[0], xs[1], got[1])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_tokens(gpu):
    x = make(0, 4, 64, "bf16", 1, gpu)
    w = make(1, 1, 64, "bf16", 2, gpu).view(64)
    pos, freq = rotation(0, 64, 3, gpu)
    hip_lib.rope(x, pos, freq, torch.empty_like(x))
    dw = [torch.full((64,), 7.0, device=gpu) for _ in "qk"]
    rstd = torch.empty((0, 8), device=gpu)
    hip_lib.qk_norm_rope_fwd(x, x, w, w, pos, freq, torch.empty_like(x), torch.empty_like(x), rstd)
    hip_lib.qk_norm_rope_bwd(x, x, w, w, pos, freq, rstd, x, x, torch.empty_like(x),
                             torch.empty_like(x), *dw)
    assert all((d == 0).all() for d in dw)
