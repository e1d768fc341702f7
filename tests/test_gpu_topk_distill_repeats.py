"""credit_topk_distill_fwd where entries name one column more than once: the KL
of their sum, against the definition over dense rows in 64 bits."""
import math

import numpy as np
import pytest
import torch

from credit_amd import hip_lib
from tests import distill_definition as definition
from tests.logits_cases import DTYPES, EPS, as64, assert_within, generator, make_logits, sum_error
from tests.test_gpu_topk_distill import forward

pytestmark = pytest.mark.gpu


def check(gpu, z, ids, teacher, tail, temperature=1.0, cfg=None, what=""):
    want = definition.loss(z, ids, teacher, tail, temperature).numpy()
    loss, _ = forward(z.to(gpu), ids, teacher, tail, temperature, gpu, cfg)
    with np.errstate(all="ignore"):
        live = ids.numpy() >= 0
        mass = np.where(live, np.exp(as64(teacher)), 0).sum(1) if tail else 1.0
    # ln p and ln of the tail by S's relative error, weighed by q; the rest in 64 bits.
    bound = 2 * sum_error(z.shape[1]) * np.maximum(1.0, mass) + np.abs(want) * EPS
    assert_within(as64(loss), want, bound, what)
    return loss


def entries(rows, cols, k, tail, seed):
    g = generator(seed)
    ids = torch.randint(0, cols, (rows, k), generator=g)
    teacher = torch.randn((rows, k), generator=g)
    return ids, torch.log_softmax(teacher, 1) - 0.25 if tail else teacher


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols,k", [(1, 2), (4, 3), (40, 64), (300, 256), (9001, 256), (50001, 17),
                                    (300007, 256)])
def test_repeats(gpu, cols, k, dtype, tail):
    """Random columns (many or few meet), one column alone, a pair, a triple of
    which one is without mass, every column twice with absent ones between."""
    print(f"topk_distill repeats {dtype} {cols} k {k} tail {tail}", flush=True)
    z = make_logits(6, cols, dtype, 331)
    ids, teacher = entries(6, cols, k, tail, 332)
    ids[1] = cols // 2
    if cols >= k:
        ids[2:] = torch.stack([torch.randperm(cols, generator=generator(i))[:k] for i in range(4)])
    ids[2, -1] = ids[2, 0]
    ids[3, [k // 2, -1]] = ids[3, 0].clone()
    teacher[3, k // 2] = -math.inf
    ids[4, 1::2] = ids[4, 0:2 * (k // 2):2].clone()
    ids[5, ::3] = -1
    ids[5, -1] = ids[5, 1]
    for variant, parts in (("read", 0), ("split", 3)):
        check(gpu, z, ids, teacher, tail, 1.3, hip_lib.make_cfg(variant, parts),
              f"{variant} {cols} {k}")


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("apart", [0, 1, 32, 4096, 65536, 131072, 262144])
def test_columns_far_apart_are_no_repeats(gpu, apart, tail):
    """Columns whose numbers differ in high bits alone; 0: the same one."""
    cols, k = 300007, 9
    print(f"topk_distill columns {apart} apart tail {tail}", flush=True)
    z = make_logits(2, cols, "f32", 333)
    ids, teacher = entries(2, cols, k, tail, 334)
    ids[:, 0] = torch.tensor([5, 37000])
    ids[:, 4] = ids[:, 0] + apart
    check(gpu, z, ids, teacher, tail)


@pytest.mark.parametrize("tail", [False, True])
def test_a_split_column_is_the_column(gpu, tail):
    """The mass of one entry dealt to as many as a row takes: the same loss."""
    cols = 20003
    print(f"topk_distill one column in 256 entries tail {tail}", flush=True)
    z = make_logits(3, cols, "bf16", 335)
    one = torch.tensor([[17], [9000], [20002]])
    t = torch.full((3, 1), math.log(0.5) if tail else 2.0)
    many = t.repeat(1, 256) - (math.log(256) if tail else 0.0)
    whole = check(gpu, z, one, t, tail)
    dealt = check(gpu, z, one.repeat(1, 256), many, tail)
    # 256 e^(t - ln 256) by the rounding of that exponent, 2^-22 of it, in q (ln q - ln p).
    assert torch.allclose(whole, dealt, rtol=1e-5, atol=1e-5)
    assert tail or (whole > 0).all()
