"""That the bounds of tests/logits_bounds.py tell apart what they are meant to:
an fp32 emulation of a gradient formed through the teacher's rounded log-sum lies
outside them, one formed about the teacher's maximum within.  No GPU."""
import numpy as np
import torch

from tests import distill_definition as definition
from tests.logits_bounds import (distill_gradient_bound, entropy_error, logprob_gradient_bound,
                                 stats, sum_error)
from tests.logits_cases import as64, generator, make_logits


def far_teacher(cols, rows=64, k=8):
    """A teacher whose logits lie near 24, at T = 0.7, and a student that gives its
    columns a share of 10^-5 or less: what is left of the gradient is q."""
    g = generator(371)
    z = make_logits(rows, cols, "f32", 372)
    ids = torch.stack([torch.randperm(cols, generator=g)[:k] for _ in range(rows)])
    z.scatter_(1, ids, -12.0)
    teacher = 24.0 + torch.randn((rows, k), generator=g)
    return z, ids, teacher, float(np.float32(0.7))


def emulated(z, ids, teacher, temperature, through_log_sum):
    """p - q with q as fp32 forms it; p exact."""
    p = torch.softmax(z.double() / temperature, 1)
    t = np.float32(temperature)
    x = teacher.numpy()
    m = x.max(1, keepdims=True)
    if through_log_sum:
        total = np.exp((as64(teacher) - m) / temperature).sum(1, keepdims=True)
        lse = np.float32(m.astype(np.float64) / temperature + np.log(total))
        q = np.exp(x / t - lse)
    else:
        e = np.exp((x - m) / t)
        q = e / e.sum(1, keepdims=True, dtype=np.float32)
    assert q.dtype == np.float32
    return p.scatter_add(1, ids, -torch.from_numpy(q).double()).div(temperature).numpy()


def test_a_rounded_log_sum_lies_outside():
    z, ids, teacher, temperature = far_teacher(300)
    dloss = torch.ones(len(z))
    want = definition.gradient(z, ids, teacher, dloss, False, temperature).numpy()
    bound = distill_gradient_bound(as64(z), ids, as64(teacher), as64(dloss), False, temperature)
    assert (np.abs(emulated(z, ids, teacher, temperature, False) - want) <= bound).all()
    wrong = np.abs(emulated(z, ids, teacher, temperature, True) - want) > bound
    assert wrong.sum() > 10


def test_the_bounds_are_small():
    """A few 10^-6 of p in rows of 4099 columns, where p is largest."""
    z = as64(make_logits(8, 4099, "f32", 373))
    st = stats(z, 1.0)
    assert (sum_error(st) < 3e-6).all() and (entropy_error(st) < 3e-5).all()
    tokens = np.full((8, 1), -1)
    tokens[:, 0] = 5
    bound = logprob_gradient_bound(z, tokens, np.ones((8, 1)), None, 1.0)
    top = z.argmax(1)[:, None]
    share = np.take_along_axis(st["p"], top, 1)
    assert (np.take_along_axis(bound, top, 1) < 4e-6 * share + 8 * 2.0 ** -24).all()
