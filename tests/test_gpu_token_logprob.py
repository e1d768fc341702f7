"""credit_token_logprob_fwd / _bwd against the oracle in 64 bits: widths and
alignments around the vectors, batches and parts a row is cut into, rows that a
mask empties, ties, padding, rows apart in memory, gradients in place."""
import math

import numpy as np
import pytest
import torch

from credit_amd import hip_lib
from oracle import reference as ref
from tests.logits_cases import (DTYPES, EPS, as64, assert_within, entropy_error, generator,
                                half_step, make_logits, placed, special_rows, sum_error)

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (3, 2), (2, 7), (5, 63), (4, 257), (3, 1000), (2, 4099), (3, 8192), (2, 8193),
          (2, 16383), (7, 20003), (2, 50001), (1, 131072), (2, 262144), (2, 300007),
          (1, 1100001), (300, 515)]


def forward(z, tokens, top, entropy=True, temperature=1.0, cfg=None):
    rows, cols = z.shape
    f32 = dict(device=z.device, dtype=torch.float32)
    logp = torch.full(tokens.shape, 7.0, **f32)
    stats = torch.full((rows, 2), 7.0, **f32)
    h = torch.full((rows,), 7.0, **f32) if entropy else None
    top_logp = torch.full((rows, top), 7.0, **f32) if top else None
    ids = torch.full((rows, top), -7, device=z.device, dtype=torch.int64) if top else None
    hip_lib.token_logprob_fwd(z, tokens.to(z.device), logp, stats, h, top_logp, ids, temperature,
                              cfg)
    torch.cuda.synchronize()
    return logp, stats, h, top_logp, ids


def check_forward(z, tokens, top, got, temperature=1.0, what=""):
    logp, stats, h, top_logp, ids = got
    cols = z.shape[1]
    e_logp, e_stats, e_h, e_top, e_ids = ref.token_logprob_fwd(as64(z), tokens.numpy(), top,
                                                               temperature)
    # ln S is off by S's relative error; the result is rounded once.
    err = sum_error(cols)
    with np.errstate(invalid="ignore"):
        assert_within(as64(logp), e_logp, err + np.abs(e_logp) * EPS, what + " logp")
        m = as64(stats)[:, 0]
        assert np.array_equal(m, e_stats[:, 0], equal_nan=True), what + " max"
        assert_within(as64(stats)[:, 1], e_stats[:, 1], e_stats[:, 1] * (err + EPS), what + " sum")
        if h is not None:
            assert_within(as64(h), e_h, entropy_error(cols) + np.abs(e_h) * EPS, what + " entropy")
        if top:
            assert np.array_equal(ids.cpu().numpy(), e_ids), what + " columns"
            assert_within(as64(top_logp), e_top, err + np.abs(e_top) * EPS, what + " top")


def random_tokens(rows, cols, n, seed):
    tokens = torch.randint(0, cols, (rows, n), generator=generator(seed))
    if n > 1:
        tokens[0, 1] = tokens[0, 0]
        tokens[-1, -1] = -100
    return tokens


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(gpu, rows, cols, dtype):
    print(f"token_logprob_fwd {dtype} {rows}x{cols}", flush=True)
    z = make_logits(rows, cols, dtype, 11)
    tokens = random_tokens(rows, cols, 3, 12)
    top = min(cols, 20)
    got = forward(z.to(gpu), tokens, top, temperature=0.7)
    check_forward(z, tokens, top, got, 0.7)


@pytest.mark.parametrize("top", [0, 1, 2, 64, 255, 256])
@pytest.mark.parametrize("entropy", [False, True])
def test_forward_options(gpu, top, entropy):
    print(f"token_logprob_fwd top {top} entropy {entropy}", flush=True)
    for dtype in DTYPES:
        z = make_logits(6, 9001, dtype, 13)
        for n in (0, 1, 256):
            tokens = random_tokens(6, 9001, n, 14) if n else torch.zeros((6, 0), dtype=torch.int64)
            check_forward(z, tokens, top, forward(z.to(gpu), tokens, top, entropy),
                          what=f"{dtype} {n} tokens")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [5, 300, 4099, 20001])
@pytest.mark.parametrize("temperature", [1.0, 0.25, 8.0])
def test_forward_special_rows(gpu, cols, dtype, temperature):
    print(f"token_logprob_fwd special rows {dtype} {cols}", flush=True)
    z, names = special_rows(cols, dtype, 15)
    tokens = torch.tensor([[0, cols // 2, cols - 1, -1, cols, 1 << 40, -(1 << 62)]] * len(names))
    top = min(cols, 40)
    got = forward(z.to(gpu), tokens, top, temperature=temperature)
    for i, name in enumerate(names):
        check_forward(z[i:i + 1], tokens[i:i + 1], top, [t[i:i + 1] for t in got], temperature,
                      name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,gap", [(0, 1), (1, 0), (3, 5), (8, 8), (7, 57)])
def test_forward_rows_apart(gpu, dtype, offset, gap):
    """Rows at any element address, NaN around them."""
    for rows, cols in ((4, 33), (3, 8191), (2, 30011)):
        print(f"token_logprob_fwd {dtype} {rows}x{cols} offset {offset} gap {gap}", flush=True)
        z = make_logits(rows, cols, dtype, 16)
        tokens = random_tokens(rows, cols, 2, 17)
        got = forward(placed(z, gpu, offset, gap), tokens, 9)
        check_forward(z, tokens, 9, got)


# ---------------------------------------------------------------- backward --


def gradient_bound(z, tokens, dlogp, dent, temperature, dtype, want):
    """e^x has 2 EPS and 3 EPS ln 2 |x| (|x| <= 126 bits: 2.7e-5/2), S its sum's
    error twice (the forward's and its rounding); the weight G + h (ln p + H) a
    few roundings and the entropy's error; a token's gradient is one sum.  An
    exponential below fp32's least normal, 2^-126, is 0: off by at most that
    times the weight (S >= 1)."""
    _, _, lp = ref._log_softmax(as64(z), temperature)
    err = 1.7e-5 + 2 * sum_error(z.shape[1])
    with np.errstate(all="ignore"):
        p = np.where(lp == -np.inf, 0.0, np.exp(lp))
        live = as64(tokens) >= 0
        weight = np.abs(as64(dlogp) * live).sum(1, keepdims=True)
        if dent is not None:
            h = np.abs(as64(dent))[:, None]
            ent = -np.where(p == 0, 0.0, p * lp).sum(1, keepdims=True)
            weight = weight + h * (np.abs(np.where(p == 0, 0.0, lp)) + ent
                                   + entropy_error(z.shape[1]) / err)
        one = np.zeros(z.shape)
        for r in range(z.shape[0]):
            for t, g in zip(tokens[r].tolist(), as64(dlogp)[r]):
                if 0 <= t < z.shape[1]:
                    one[r, t] += abs(g)
        bound = (p * weight * err + one * 8 * EPS + 2.0 ** -126 * (weight + 1)) / temperature
        return bound + np.abs(want) * half_step(dtype) * (1 + 1e-6)


def backward(z, tokens, dlogp, dent, temperature, gpu, out=None, cfg=None):
    _, stats, h, _, _ = forward(z, tokens, 0, dent is not None, temperature)
    out = torch.full(z.shape, 7.0, dtype=z.dtype, device=gpu) if out is None else out
    hip_lib.token_logprob_bwd(z, tokens.to(gpu), stats, dlogp.to(gpu), out, h,
                              None if dent is None else dent.to(gpu), temperature, cfg)
    torch.cuda.synchronize()
    return out


def check_backward(z, tokens, dlogp, dent, temperature, dtype, out, what=""):
    want = ref.token_logprob_bwd(as64(z), tokens.numpy(), as64(dlogp),
                                 None if dent is None else as64(dent), temperature)
    bound = gradient_bound(z, tokens, dlogp, dent, temperature, dtype, want)
    assert_within(as64(out), want, bound, what + " dlogits")


@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_backward(gpu, rows, cols, dtype, entropy):
    print(f"token_logprob_bwd {dtype} {rows}x{cols} entropy {entropy}", flush=True)
    g = generator(21)
    z = make_logits(rows, cols, dtype, 22)
    tokens = random_tokens(rows, cols, 3, 23)
    dlogp = torch.randn(tokens.shape, generator=g)
    dent = torch.randn(rows, generator=g) if entropy else None
    out = backward(z.to(gpu), tokens, dlogp, dent, 0.7, gpu)
    check_backward(z, tokens, dlogp, dent, 0.7, dtype, out)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [5, 300, 20001])
def test_backward_special_rows(gpu, cols, dtype):
    print(f"token_logprob_bwd special rows {dtype} {cols}", flush=True)
    z, names = special_rows(cols, dtype, 24)
    g = generator(25)
    tokens = torch.tensor([[0, cols // 2, cols // 2, cols - 1]] * len(names))
    dlogp = torch.randn(tokens.shape, generator=g)
    dent = torch.randn(len(names), generator=g)
    out = backward(z.to(gpu), tokens, dlogp, dent, 1.0, gpu)
    for i, name in enumerate(names):
        s = slice(i, i + 1)
        check_backward(z[s], tokens[s], dlogp[s], dent[s], 1.0, dtype, out[s], name)


@pytest.mark.parametrize("dtype", DTYPES)
def test_backward_padding_is_zero_whatever_the_row_holds(gpu, dtype):
    print(f"token_logprob_bwd padding {dtype}", flush=True)
    rows, cols = 6, 9001
    z = make_logits(rows, cols, dtype, 26).to(gpu)
    z[2:] = math.nan
    tokens = torch.randint(0, cols, (rows, 2), generator=generator(27))
    dlogp = torch.ones((rows, 2))
    tokens[2] = -1                       # padding alone
    dlogp[3] = 0.0                       # weights of 0
    tokens[4, 0], dlogp[4, 1] = -5, 0.0  # one of each
    dent = torch.ones(rows)
    dent[2:5] = 0.0
    out = backward(z, tokens, dlogp, dent, 1.0, gpu)
    assert (out[2:5] == 0).all() and torch.isnan(out[5]).all()
    check_backward(z[:2].cpu(), tokens[:2], dlogp[:2], dent[:2], 1.0, dtype, out[:2])
    # A column that is none: its row is NaN, unless its weight is 0.
    tokens[0, 0], tokens[1, 1], dlogp[1, 1] = cols, 1 << 33, 0.0
    out = backward(z, tokens, dlogp, None, 1.0, gpu)
    assert torch.isnan(out[0]).all()
    check_backward(z[1:2].cpu(), tokens[1:2], dlogp[1:2], None, 1.0, dtype, out[1:2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("zo,zg,do,dg", [(0, 0, 0, 3), (1, 0, 0, 0), (3, 5, 3, 5), (2, 6, 10, 14),
                                         (0, 8, 0, 0)])
def test_backward_rows_apart(gpu, dtype, zo, zg, do, dg):
    """In and out at different offsets and distances; what lies between the
    rows of the gradient is left as it was."""
    for rows, cols in ((4, 33), (3, 8191), (2, 30011)):
        print(f"token_logprob_bwd {dtype} {rows}x{cols} {zo, zg, do, dg}", flush=True)
        z = make_logits(rows, cols, dtype, 28)
        tokens = random_tokens(rows, cols, 2, 29)
        dlogp = torch.randn(tokens.shape, generator=generator(30))
        flat = torch.full((do + rows * (cols + dg) + 9,), 3.0, dtype=DTYPES[dtype], device=gpu)
        out = flat[do:do + rows * (cols + dg)].view(rows, cols + dg)
        zs = placed(z, gpu, zo, zg)
        _, stats, _, _, _ = forward(zs, tokens, 0, False)
        hip_lib.token_logprob_bwd(zs, tokens.to(gpu), stats, dlogp.to(gpu), out[:, :cols])
        torch.cuda.synchronize()
        check_backward(z, tokens, dlogp, None, 1.0, dtype, out[:, :cols])
        assert (out[:, cols:] == 3).all() and (flat[:do] == 3).all() and (flat[-9:] == 3).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [100, 8193, 40003])
def test_backward_in_place(gpu, dtype, cols):
    """The gradient over the logits themselves: the same bits."""
    print(f"token_logprob_bwd in place {dtype} {cols}", flush=True)
    rows = 5
    z = make_logits(rows, cols, dtype, 31).to(gpu)
    tokens = random_tokens(rows, cols, 40, 32)
    dlogp = torch.randn(tokens.shape, generator=generator(33))
    dent = torch.randn(rows, generator=generator(34))
    apart = backward(z, tokens, dlogp, dent, 1.3, gpu)
    over = z.clone()
    backward(over, tokens, dlogp, dent, 1.3, gpu, out=over)
    assert torch.equal(apart, over)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols,offset", [(256, 0), (300, 5), (9001, 1), (131072, 0)])
def test_backward_crowded_tokens(gpu, dtype, cols, offset):
    """As many tokens as a row takes: neighbours, all of them one, the row's ends."""
    print(f"token_logprob_bwd crowded {dtype} {cols}", flush=True)
    z = make_logits(4, cols, dtype, 51)
    tokens = torch.randint(0, cols, (4, 256), generator=generator(52))
    tokens[0] = cols - 256 + torch.arange(256)
    tokens[1] = cols // 2
    tokens[2] = torch.arange(256) // 2 * 2
    dlogp = torch.randn(tokens.shape, generator=generator(53))
    dent = torch.randn(4, generator=generator(54))
    apart = backward(placed(z, gpu, offset, offset), tokens, dlogp, dent, 0.9, gpu)
    check_backward(z, tokens, dlogp, dent, 0.9, dtype, apart)
    over = placed(z, gpu, offset, offset)
    backward(over, tokens, dlogp, dent, 0.9, gpu, out=over)
    assert torch.equal(apart, over)


def test_backward_against_differences(gpu):
    """The kernels' own forward, differentiated numerically."""
    rows, cols, step = 3, 37, 1e-2
    z = make_logits(rows, cols, "f32", 35)
    tokens = random_tokens(rows, cols, 2, 36)
    dlogp = torch.randn(tokens.shape, generator=generator(37))
    dent = torch.randn(rows, generator=generator(38))
    out = as64(backward(z.to(gpu), tokens, dlogp, dent, 1.0, gpu))

    def value(zz):
        logp, _, h, _, _ = forward(zz.to(gpu), tokens.repeat(cols, 1), 0)
        live = (tokens >= 0).repeat(cols, 1)
        per_row = (logp.cpu().double() * live * dlogp.double().repeat(cols, 1)).sum(1)
        return (per_row + h.cpu().double() * dent.double().repeat(cols)).view(cols, rows).t()

    eye = torch.eye(cols)[:, None, :] * step
    up, down = ((z[None] + s * eye).reshape(cols * rows, cols) for s in (1, -1))
    numeric = ((value(up) - value(down)) / (2 * step)).numpy()
    # Differences: the third derivative (at most 6 |weights|) times step^2 / 6,
    # and the forward's errors over the step.
    w = (np.abs(as64(dlogp)).sum(1) + 20 * np.abs(as64(dent)))[:, None]
    bound = w * (step ** 2 + (sum_error(cols) + entropy_error(cols)) / step)
    assert_within(out, numeric, bound, "differences")


@pytest.mark.parametrize("dtype", DTYPES)
def test_alternatives_that_crowd(gpu, dtype):
    """The largest values side by side, in one lane's vectors, or too many equal
    ones for any list."""
    cols = 70001
    z = make_logits(6, cols, dtype, 42)
    g = generator(43)
    z[0, 100:400] = torch.rand(300, generator=g).to(z.dtype) + 30
    lane = torch.arange(0, cols - 8192, 8192)[:, None] + torch.arange(4)  # one lane's columns
    z[1, lane.flatten()] = (torch.rand(lane.numel(), generator=g) + 30).to(z.dtype)
    z[2, ::7] = 25.0
    z[3, 5000:5000 + 1500] = torch.linspace(20, 40, 1500).to(z.dtype)
    z[4] = z[4].clamp(max=2.0)
    z[5, 64:] = -math.inf
    tokens = random_tokens(6, cols, 1, 44)
    for top in (1, 30, 64, 200, 256):
        print(f"token_logprob_fwd crowd {dtype} top {top}", flush=True)
        check_forward(z, tokens, top, forward(z.to(gpu), tokens, top), what=f"top {top}")


def masked_rows(cols, dtype, seed):
    """Rows of which a mask leaves little, at random columns, in one place, or
    behind everything else; equal values in few or all places."""
    g = generator(seed)
    low = torch.finfo(DTYPES[dtype]).min
    base = make_logits(1, cols, dtype, seed + 1)[0]
    rows = []
    for fill in (-math.inf, low, -4.0):
        for n in (0, 1, 10, 100, 1500):
            z = torch.full((cols,), fill)
            at = torch.randperm(cols, generator=g)[:n]
            z[at] = base[at].float().abs()
            rows.append(z)
    rows.append(torch.full((cols,), -math.inf).index_fill(0, torch.arange(cols - 70, cols), 2.0))
    rows.append(torch.where(torch.arange(cols) < cols - 9, 1.0, -1.0).index_fill(
        0, torch.tensor([cols // 2]), 3.0))
    rows.append(torch.where(torch.arange(cols) < cols - 300, low, 0.0))
    rows.append(torch.full((cols,), math.inf))
    rows.append(torch.full((cols,), -math.inf).index_fill(0, torch.arange(5, cols, 97), -0.0)
                .index_fill(0, torch.arange(7, cols, 97), 0.0))
    rows.append(torch.full((cols,), math.nan).index_fill(0, torch.arange(0, cols, 2), -math.inf))
    return torch.stack(rows).to(DTYPES[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("variant", ["read", "split"])
@pytest.mark.parametrize("cols,offset", [(300, 0), (5003, 3), (70001, 1), (131072, 0)])
def test_alternatives_of_masked_rows(gpu, dtype, variant, cols, offset):
    z = masked_rows(cols, dtype, 49)
    tokens = torch.randint(0, cols, (len(z), 2), generator=generator(50))
    cfg = hip_lib.make_cfg(variant, 5 if variant == "split" else 0)
    zs = placed(z, gpu, offset, offset)
    for top in (1, 2, 20, 101, 256):
        print(f"token_logprob masked {dtype} {variant} {cols} top {top}", flush=True)
        check_forward(z, tokens, top, forward(zs, tokens, top, cfg=cfg), what=f"top {top}")


def test_more_rows_than_a_grid_has(gpu):
    rows, cols = 70001, 5
    print("token_logprob many rows", flush=True)
    z = make_logits(rows, cols, "f32", 45)
    tokens = torch.randint(0, cols, (rows, 1), generator=generator(46))
    check_forward(z, tokens, 3, forward(z.to(gpu), tokens, 3))
    dlogp = torch.randn(tokens.shape, generator=generator(47))
    out = backward(z.to(gpu), tokens, dlogp, None, 1.0, gpu)
    want = torch.autograd.functional.vjp(
        lambda x: torch.log_softmax(x, 1).gather(1, tokens), z.double(), dlogp.double())[1]
    p = torch.softmax(z.double(), 1).numpy()
    one = torch.zeros(z.shape, dtype=torch.float64).scatter_(1, tokens, dlogp.double().abs())
    bound = p * dlogp.double().abs().numpy() * (1.7e-5 + 2 * sum_error(cols))
    bound += one.numpy() * 8 * EPS
    assert_within(as64(out), want.numpy(), bound, "dlogits")


def test_more_threads_than_a_grid_has(gpu):
    """2^24 workgroups have 2^32 threads: more rows than that, each as it is in
    a call of its own."""
    rows, cols = (1 << 24) + 5, 2
    print("token_logprob 2^24 rows", flush=True)
    z = torch.randn((rows, cols), generator=generator(48)).to(gpu)
    tokens = torch.arange(rows, device=gpu).remainder(3)[:, None] - 1
    got = forward(z, tokens, 1)
    for s in (slice(0, 100), slice((1 << 23) - 50, (1 << 23) + 50), slice(rows - 100, rows)):
        alone = forward(z[s], tokens[s], 1)
        for a, b in zip(got, alone):
            assert torch.equal(a[s], b)
        check_forward(z[s].cpu(), tokens[s].cpu(), 1, alone)
    assert not (got[0] == 7.0).any() and not (got[4] == -7).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("variant", ["read", "split"])
def test_lowest_values_ahead_of_a_far_maximum(gpu, dtype, variant):
    """A lane's first batches hold the type's lowest values alone, later ones
    values beyond 2^20: from one to the other is further than fp32 goes."""
    cols = 5 * 8192 + 77
    print(f"token_logprob far maximum {dtype} {variant}", flush=True)
    z = torch.full((3, cols), torch.finfo(DTYPES[dtype]).min)
    z[0, 2 * 8192:] = 2.0 ** 22
    z[1, 4 * 8192 + 5] = 2.0 ** 100
    z[1, 4 * 8192 + 3000:] = -2.0 ** 100
    z[2, 3 * 8192:] = 2.0 ** 23 + 2.0 ** 15 * (torch.arange(cols - 3 * 8192) % 3)
    z = z.to(DTYPES[dtype])
    tokens = torch.tensor([[0, cols - 1], [4 * 8192 + 5, 1], [cols - 2, cols - 3]])
    cfg = hip_lib.make_cfg(variant, 3 if variant == "split" else 0)
    check_forward(z, tokens, 9, forward(z.to(gpu), tokens, 9, cfg=cfg))


def test_offsets_beyond_32_bits(gpu):
    """Rows whose elements lie more than 2^32 bytes and 2^31 elements into the
    logits."""
    rows, cols, ld = 5, 70001, (1 << 29) + 9
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    flat = torch.empty((rows - 1) * ld + cols, dtype=torch.bfloat16, device=gpu)
    zs = torch.as_strided(flat, (rows, cols), (ld, 1))
    z = make_logits(rows, cols, "bf16", 39)
    zs.copy_(z)
    tokens = random_tokens(rows, cols, 2, 40)
    print("token_logprob far rows", flush=True)
    check_forward(z, tokens, 7, forward(zs, tokens, 7))
    dlogp = torch.randn(tokens.shape, generator=generator(41))
    backward(zs, tokens, dlogp, None, 1.0, gpu, out=zs)
    check_backward(z, tokens, dlogp, None, 1.0, "bf16", zs)
