"""credit_topk_distill_fwd / _bwd against the oracle in 64 bits: both kinds of
teacher, absent and repeated entries, rows that a mask empties, tails too small
for 1 - sum p, rows apart in memory, gradients in place."""
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from credit_amd import hip_lib
from oracle import reference as ref
from tests.logits_cases import (DTYPES, EPS, as64, assert_within, generator, half_step,
                                make_logits, placed, special_rows, sum_error)

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 63, 64), (4, 257, 9), (3, 1000, 256), (2, 4099, 20),
          (3, 8192, 31), (2, 8193, 100), (7, 20003, 64), (2, 50001, 5), (1, 131072, 64),
          (2, 262144, 128), (300, 515, 17), (2, 300007, 33)]


def make_teacher(z, k, tail, temperature, seed, noise=0.7):
    """The k largest of a teacher near z (fewer columns: the rest absent)."""
    g = generator(seed)
    rows, cols = z.shape
    t = torch.where(torch.isfinite(z.double()), z.double(), 0.0).clamp(-30, 30)
    t = t + noise * torch.randn(z.shape, generator=g, dtype=torch.float64)
    values, ids = t.topk(min(k, cols), dim=1)
    if tail:
        values = values / temperature - torch.logsumexp(t / temperature, 1, keepdim=True)
    if k > cols:
        ids = F.pad(ids, (0, k - cols), value=-1)
        values = F.pad(values, (0, k - cols), value=0.5)
    return ids.contiguous(), values.float().contiguous()


def forward(z, ids, teacher, tail, temperature, gpu, cfg=None):
    loss = torch.full((z.shape[0],), 7.0, device=gpu)
    stats = torch.full((z.shape[0], 8), 7.0, device=gpu)
    hip_lib.topk_distill_fwd(z, ids.to(gpu), teacher.to(gpu), loss, stats, tail, temperature, cfg)
    torch.cuda.synchronize()
    return loss, stats


def check_loss(z, ids, teacher, tail, temperature, loss, what=""):
    """ln p and ln of the tail are off by S's relative error, each weighed by
    its q (their sum is near 1, or what the teacher's entries sum to)."""
    want = ref.topk_distill_fwd(as64(z), ids.numpy(), as64(teacher), tail, temperature)
    with np.errstate(all="ignore"):
        mass = np.where(ids.numpy() >= 0, np.exp(as64(teacher)), 0).sum(1) if tail else 1.0
    bound = 2 * sum_error(z.shape[1]) * np.maximum(1.0, mass) + np.abs(want) * EPS
    assert_within(as64(loss), want, bound, what + " loss")


def backward(z, ids, teacher, dloss, tail, temperature, gpu, out=None, cfg=None):
    _, stats = forward(z, ids, teacher, tail, temperature, gpu)
    out = torch.full(z.shape, 7.0, dtype=z.dtype, device=gpu) if out is None else out
    hip_lib.topk_distill_bwd(z, ids.to(gpu), teacher.to(gpu), stats, dloss.to(gpu), out, tail,
                             temperature, cfg)
    torch.cuda.synchronize()
    return out


def check_gradient(z, ids, teacher, dloss, tail, temperature, dtype, out, what=""):
    """Q p and q (or the rest's share) each off by a relative error: that of an
    exponential (|x| <= 126 bits: 1.7e-5), of the sums (S, the tail's) and a few
    roundings; a tail's two terms share one exponential.  An exponential below
    fp32's least normal, 2^-126, is 0."""
    args = (as64(z), ids.numpy(), as64(teacher))
    want = ref.topk_distill_bwd(*args, as64(dloss), tail, temperature)
    p_only = np.exp(ref._log_softmax(as64(z), temperature)[2])
    g = np.abs(as64(dloss))[:, None] / temperature
    with np.errstate(all="ignore"):
        q = np.abs(want) / np.where(g == 0, 1, g) + 3 * p_only  # >= Q p + q up to Q = 2
        bound = g * q * (1.7e-5 + 4 * sum_error(z.shape[1])) + 2.0 ** -126 * (4 * g + 1)
        bound = bound + np.abs(want) * half_step(dtype) * (1 + 1e-6)
    assert_within(as64(out), want, bound, what + " dlogits")


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,k", SHAPES)
def test_loss_and_gradient(gpu, rows, cols, k, dtype, tail):
    print(f"topk_distill {dtype} {rows}x{cols} k {k} tail {tail}", flush=True)
    z = make_logits(rows, cols, dtype, 51)
    ids, teacher = make_teacher(z, k, tail, 1.5, 52)
    loss, stats = forward(z.to(gpu), ids, teacher, tail, 1.5, gpu)
    check_loss(z, ids, teacher, tail, 1.5, loss)
    m, total, _ = ref._log_softmax(as64(z), 1.5)
    assert np.array_equal(as64(stats)[:, 0], m[:, 0])
    assert_within(as64(stats)[:, 1], total[:, 0], total[:, 0] * (sum_error(cols) + EPS), "sum")
    dloss = torch.randn(rows, generator=generator(53))
    out = backward(z.to(gpu), ids, teacher, dloss, tail, 1.5, gpu)
    check_gradient(z, ids, teacher, dloss, tail, 1.5, dtype, out)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [5, 300, 20001])
def test_special_rows(gpu, cols, dtype, tail):
    print(f"topk_distill special rows {dtype} {cols} tail {tail}", flush=True)
    z, names = special_rows(cols, dtype, 54)
    ids, teacher = make_teacher(z, min(cols, 9), tail, 1.0, 55)
    dloss = torch.randn(len(names), generator=generator(56))
    loss, _ = forward(z.to(gpu), ids, teacher, tail, 1.0, gpu)
    out = backward(z.to(gpu), ids, teacher, dloss, tail, 1.0, gpu)
    for i, name in enumerate(names):
        s = slice(i, i + 1)
        check_loss(z[s], ids[s], teacher[s], tail, 1.0, loss[s], name)
        check_gradient(z[s], ids[s], teacher[s], dloss[s], tail, 1.0, dtype, out[s], name)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_absent_and_repeated_entries(gpu, dtype, tail):
    print(f"topk_distill entries {dtype} tail {tail}", flush=True)
    rows, cols, k = 9, 9001, 12
    z = make_logits(rows, cols, dtype, 57)
    ids, teacher = make_teacher(z, k, tail, 1.0, 58)
    if tail:
        teacher -= 1.0                 # room for what is added below
    ids[0, 3:] = -1
    ids[1, ::2] = -9
    ids[2] = -1                        # no entry at all
    ids[3, 5] = ids[3, 2]              # one column named twice
    ids[4, :] = ids[4, 0]              # and by every entry
    teacher[4] -= 4.0 if tail else 0.0
    teacher[5, 1:] = -math.inf         # teacher mass 0
    teacher[6] = -math.inf             # everywhere
    ids[7, 4] = cols                   # a column that is none
    teacher[8, 0] = math.nan
    loss, stats = forward(z.to(gpu), ids, teacher, tail, 1.0, gpu)
    check_loss(z, ids, teacher, tail, 1.0, loss)
    assert loss[2] == 0 and (stats[2] == 0).all() and torch.isnan(loss[7:]).all()
    dloss = torch.randn(rows, generator=generator(59))
    out = backward(z.to(gpu), ids, teacher, dloss, tail, 1.0, gpu)
    s = slice(0, 7)
    check_gradient(z[s], ids[s], teacher[s], dloss[s], tail, 1.0, dtype, out[s])
    assert torch.isnan(out[7:]).all() and (out[2] == 0).all()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols,offset", [(256, 0), (300, 5), (9001, 1), (131072, 0)])
def test_crowded_entries(gpu, cols, offset, dtype, tail):
    """As many entries as a row takes: neighbours, most of them one column, the
    row's ends, each column twice."""
    print(f"topk_distill crowded {dtype} {cols} tail {tail}", flush=True)
    z = make_logits(4, cols, dtype, 76)
    at = torch.arange(256)
    ids = torch.stack([cols - 256 + at, torch.where(at < 3, at, cols // 2), at // 2 * 2,
                       torch.randperm(cols, generator=generator(77))[:256]])
    teacher = torch.randn(ids.shape, generator=generator(78))
    if tail:
        teacher = torch.log_softmax(teacher, 1) - 0.125
    dloss = torch.randn(4, generator=generator(79))
    zs = placed(z, gpu, offset, offset)
    loss, _ = forward(zs, ids, teacher, tail, 0.9, gpu)
    check_loss(z, ids, teacher, tail, 0.9, loss)
    apart = backward(zs, ids, teacher, dloss, tail, 0.9, gpu)
    check_gradient(z, ids, teacher, dloss, tail, 0.9, dtype, apart)
    backward(zs, ids, teacher, dloss, tail, 0.9, gpu, out=zs)
    assert torch.equal(apart, zs)


@pytest.mark.parametrize("tail", [False, True])
def test_rows_without_weight_are_not_read(gpu, tail):
    rows, cols = 4, 5003
    z = make_logits(rows, cols, "bf16", 60).to(gpu)
    ids, teacher = make_teacher(z.cpu(), 8, tail, 1.0, 61)
    z[1:3] = math.nan
    ids[1] = -1
    dloss = torch.ones(rows)
    dloss[2] = 0.0
    loss, _ = forward(z, ids, teacher, tail, 1.0, gpu)
    assert loss[1] == 0 and torch.isnan(loss[2])
    out = backward(z, ids, teacher, dloss, tail, 1.0, gpu)
    assert (out[1:3] == 0).all() and not torch.isnan(out).any()


def test_small_tails_keep_their_precision(gpu):
    """A student that leaves the tail 1e-9 or 1e-30 of its mass: 1 - sum p in
    32 bits would be 0 or noise."""
    cols = 3001
    for drop in (20.0, 60.0):
        z = make_logits(2, cols, "f32", 62)
        ids, teacher = make_teacher(z, 16, True, 1.0, 63)
        mask = torch.ones((2, cols), dtype=torch.bool).scatter_(1, ids, False)
        z = torch.where(mask, z - drop, z)
        loss, _ = forward(z.to(gpu), ids, teacher, True, 1.0, gpu)
        check_loss(z, ids, teacher, True, 1.0, loss, f"tail {drop} lower")
        dloss = torch.ones(2)
        out = backward(z.to(gpu), ids, teacher, dloss, True, 1.0, gpu)
        check_gradient(z, ids, teacher, dloss, True, 1.0, "f32", out, f"tail {drop} lower")


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("zo,zg,do,dg", [(0, 0, 0, 3), (1, 0, 0, 0), (3, 5, 3, 5), (2, 6, 10, 14)])
def test_rows_apart(gpu, dtype, tail, zo, zg, do, dg):
    for rows, cols in ((4, 33), (3, 8191), (2, 30011)):
        print(f"topk_distill {dtype} {rows}x{cols} {zo, zg, do, dg} tail {tail}", flush=True)
        z = make_logits(rows, cols, dtype, 64)
        ids, teacher = make_teacher(z, 13, tail, 1.0, 65)
        zs = placed(z, gpu, zo, zg)
        loss, stats = forward(zs, ids, teacher, tail, 1.0, gpu)
        check_loss(z, ids, teacher, tail, 1.0, loss)
        flat = torch.full((do + rows * (cols + dg) + 9,), 3.0, dtype=DTYPES[dtype], device=gpu)
        out = flat[do:do + rows * (cols + dg)].view(rows, cols + dg)
        dloss = torch.randn(rows, generator=generator(66))
        hip_lib.topk_distill_bwd(zs, ids.to(gpu), teacher.to(gpu), stats, dloss.to(gpu),
                                 out[:, :cols], tail)
        torch.cuda.synchronize()
        check_gradient(z, ids, teacher, dloss, tail, 1.0, dtype, out[:, :cols])
        assert (out[:, cols:] == 3).all() and (flat[:do] == 3).all() and (flat[-9:] == 3).all()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_in_place(gpu, dtype, tail):
    for cols in (100, 8193, 40003):
        print(f"topk_distill_bwd in place {dtype} {cols}", flush=True)
        z = make_logits(5, cols, dtype, 67)
        ids, teacher = make_teacher(z, 70, tail, 1.0, 68)
        dloss = torch.randn(5, generator=generator(69))
        apart = backward(z.to(gpu), ids, teacher, dloss, tail, 1.0, gpu)
        over = z.to(gpu)
        backward(over, ids, teacher, dloss, tail, 1.0, gpu, out=over)
        assert torch.equal(apart, over)


@pytest.mark.parametrize("tail", [False, True])
def test_more_rows_than_a_grid_has(gpu, tail):
    """Every row as it is alone: the rows beyond 65535 of one call against a
    call of their own."""
    rows, cols = 70001, 9
    print(f"topk_distill many rows tail {tail}", flush=True)
    z = make_logits(rows, cols, "f32", 72).to(gpu)
    ids, teacher = make_teacher(z.cpu(), 4, tail, 1.0, 73)
    ids[::3, 1] = ids[::3, 0]
    dloss = torch.randn(rows, generator=generator(74))
    loss, _ = forward(z, ids, teacher, tail, 1.0, gpu)
    out = backward(z, ids, teacher, dloss, tail, 1.0, gpu)
    for s in (slice(0, 100), slice(65436, 65636), slice(69901, rows)):
        alone, _ = forward(z[s], ids[s], teacher[s], tail, 1.0, gpu)
        assert torch.equal(loss[s], alone)
        assert torch.equal(out[s], backward(z[s], ids[s], teacher[s], dloss[s], tail, 1.0, gpu))
        check_loss(z[s].cpu(), ids[s], teacher[s], tail, 1.0, alone)


def test_more_threads_than_a_grid_has(gpu):
    rows, cols = (1 << 24) + 5, 2
    print("topk_distill 2^24 rows", flush=True)
    z = torch.randn((rows, cols), generator=generator(75)).to(gpu)
    ids = torch.arange(rows, device=gpu).remainder(2)[:, None].contiguous()
    teacher = torch.full((rows, 1), -0.25)
    loss, _ = forward(z, ids, teacher, True, 1.0, gpu)
    for s in (slice(0, 100), slice((1 << 23) - 50, (1 << 23) + 50), slice(rows - 100, rows)):
        alone, _ = forward(z[s], ids[s], teacher[s], True, 1.0, gpu)
        assert torch.equal(loss[s], alone)
        check_loss(z[s].cpu(), ids[s].cpu(), teacher[s], True, 1.0, alone)


def test_gradient_against_differences(gpu):
    rows, cols, step = 2, 37, 1e-2
    z = make_logits(rows, cols, "f32", 70)
    for tail in (False, True):
        ids, teacher = make_teacher(z, 6, tail, 1.0, 71)
        dloss = torch.ones(rows)
        out = as64(backward(z.to(gpu), ids, teacher, dloss, tail, 1.0, gpu))
        eye = torch.eye(cols)[:, None, :] * step
        up, down = (forward((z[None] + s * eye).reshape(cols * rows, cols).to(gpu),
                            ids.repeat(cols, 1), teacher.repeat(cols, 1), tail, 1.0,
                            gpu)[0].cpu().double().view(cols, rows).t() for s in (1, -1))
        numeric = ((up - down) / (2 * step)).numpy()
        # The third derivative of ln p is at most 6 / 6 step^2; the loss's error.
        assert_within(out, numeric, 2 * step ** 2 + 4 * sum_error(cols) / step, f"tail {tail}")
