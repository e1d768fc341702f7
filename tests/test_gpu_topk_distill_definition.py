"""credit_topk_distill_fwd / _bwd against the loss's definition over dense rows
in 64 bits: rows whose columns outside the entries have no mass."""
import math

import numpy as np
import pytest
import torch

from credit_amd import hip_lib
from tests import distill_definition as definition
from tests.logits_bounds import distill_gradient_bound, rounded
from tests.logits_cases import DTYPES, EPS, as64, assert_within, generator, make_logits, sum_error
from tests.test_gpu_topk_distill import forward

pytestmark = pytest.mark.gpu


def check(gpu, z, ids, teacher, tail, temperature, what, cfg=None):
    """Loss and gradient."""
    print(f"topk_distill {what} {z.dtype} {tuple(z.shape)}", flush=True)
    rows, cols = z.shape
    dloss = torch.linspace(-1.0, 2.0, rows)
    zg = z.to(gpu)
    loss, stats = forward(zg, ids, teacher, tail, temperature, gpu, cfg)
    want = definition.loss(z, ids, teacher, tail, temperature).numpy()
    live = ids.numpy() >= 0
    with np.errstate(all="ignore"):
        mass = np.where(live, np.exp(as64(teacher)), 0).sum(1) if tail else 1.0
    bound = 2 * sum_error(cols) * np.maximum(1.0, mass) + np.abs(want) * EPS
    assert_within(as64(loss), want, bound, what + " loss")
    out = torch.full_like(zg, 7.0)
    hip_lib.topk_distill_bwd(zg, ids.to(gpu), teacher.to(gpu), stats, dloss.to(gpu), out, tail,
                             temperature)
    torch.cuda.synchronize()
    want = definition.gradient(z, ids, teacher, dloss, tail, temperature).numpy()
    bound = distill_gradient_bound(as64(z), ids, as64(teacher), as64(dloss), tail, temperature)
    assert_within(as64(out), want, rounded(bound, want, z.dtype), what + " dlogits")


@pytest.mark.parametrize("temperature", [1.0, 0.75])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols,k", [(11, 3), (300, 40), (8001, 3)])
def test_a_tail_without_mass(gpu, cols, k, dtype, temperature):
    """Masked columns but for the entries', whose q leave mass: nothing is held
    against the others, in the gradient either."""
    g = generator(311)
    z = make_logits(5, cols, dtype, 312)
    ids = torch.stack([torch.randperm(cols, generator=g)[:k] for _ in range(5)])
    masked = torch.ones(z.shape, dtype=torch.bool).scatter_(1, ids, False)
    masked[4] = False
    z[masked] = -math.inf
    teacher = torch.log_softmax(torch.randn((5, k), generator=g), 1) - 0.25
    teacher[1] = -math.inf                      # no mass at all
    teacher[2] += 0.75                          # more than 1
    ids[3, 1:] = -1                             # one entry
    z[3] = torch.where(torch.arange(cols) == ids[3, 0], z[3].clamp(-9, 9), -math.inf)
    check(gpu, z, ids, teacher, True, temperature, "tail without mass")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [1, 5, 256])
def test_every_column_is_named(gpu, cols, dtype):
    g = generator(313)
    z = make_logits(4, cols, dtype, 314)
    ids = torch.stack([torch.randperm(cols, generator=g) for _ in range(4)])
    teacher = torch.log_softmax(torch.randn((4, cols), generator=g), 1) - 0.25
    check(gpu, z, ids, teacher, True, 2.0, "every column named")


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_tail_without_mass_in_parts(gpu, dtype):
    """Parts, most of them without any column: statistics as one workgroup's."""
    cols = 50001
    print(f"topk_distill tail without mass in parts {dtype}", flush=True)
    g = generator(315)
    z = make_logits(3, cols, dtype, 316)
    ids = torch.stack([torch.randperm(cols, generator=g)[:7] for _ in range(3)])
    z[torch.ones(z.shape, dtype=torch.bool).scatter_(1, ids, False)] = -math.inf
    teacher = torch.log_softmax(torch.randn((3, 7), generator=g), 1) - 0.25
    teacher[1] = -math.inf
    for variant, parts in (("read", 0), ("split", 3), ("split", 7)):
        loss, stats = forward(z.to(gpu), ids, teacher, True, 1.0, gpu,
                              hip_lib.make_cfg(variant, parts))
        want = definition.loss(z, ids, teacher, True)
        assert_within(as64(loss), want.numpy(), 2 * sum_error(cols) + want.abs().numpy() * EPS,
                      f"loss {variant} {parts}")
        # Q = sum q, and no gradient for the tail.
        np.testing.assert_allclose(as64(stats)[:, 4], as64(teacher.double().exp().sum(1)),
                                   rtol=2 * EPS, atol=0)
        assert (stats[:, 5] == 0).all()
