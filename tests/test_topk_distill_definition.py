"""The oracle of the distillation against its definition over dense rows, and
against differences: rows whose columns outside the entries have no mass."""
import math

import numpy as np
import pytest
import torch

from oracle import reference as ref
from tests import distill_definition as definition
from tests.logits_cases import generator

STEP = 1e-6


def rows_without_tail_mass(cols=11, k=3, seed=301):
    """(z, ids, teacher) whose columns outside the entries are all masked, with
    mass left for them; the last row is not masked."""
    g = generator(seed)
    z = torch.randn((4, cols), generator=g, dtype=torch.float64)
    ids = torch.stack([torch.randperm(cols, generator=g)[:k] for _ in range(4)])
    teacher = torch.log(torch.tensor([0.4, 0.3, 0.1], dtype=torch.float64)).repeat(4, 1)
    masked = torch.ones(z.shape, dtype=torch.bool).scatter_(1, ids, False)
    masked[-1] = False
    z[masked] = -math.inf
    teacher[1] = -math.inf      # no mass anywhere but in a tail that is not there
    teacher[2, 2] = math.log(0.9)  # more than 1
    return z, ids, teacher


def differences(z, ids, teacher, dloss, tail, temperature):
    """Of the oracle's own loss; columns of -inf stay where they are: 0."""
    z, ids, teacher = z.numpy(), ids.numpy(), teacher.numpy()
    out = np.zeros(z.shape)
    for j in range(z.shape[1]):
        up, down = z.copy(), z.copy()
        up[:, j] += STEP
        down[:, j] -= STEP
        out[:, j] = (ref.topk_distill_fwd(up, ids, teacher, tail, temperature)
                     - ref.topk_distill_fwd(down, ids, teacher, tail, temperature)) / (2 * STEP)
    return out * dloss.numpy()[:, None]


def check(z, ids, teacher, tail, temperature):
    dloss = torch.linspace(-1.0, 2.0, z.shape[0], dtype=torch.float64)
    np.testing.assert_allclose(
        ref.topk_distill_fwd(z.numpy(), ids.numpy(), teacher.numpy(), tail, temperature),
        definition.loss(z, ids, teacher, tail, temperature).numpy(), rtol=1e-12, atol=1e-13)
    got = ref.topk_distill_bwd(z.numpy(), ids.numpy(), teacher.numpy(), dloss.numpy(), tail,
                               temperature)
    np.testing.assert_allclose(
        got, definition.gradient(z, ids, teacher, dloss, tail, temperature).numpy(), atol=1e-12)
    # The loss's third derivative times STEP^2 / 6, and 2^-52 of a loss over STEP.
    numeric = differences(z, ids, teacher, dloss, tail, temperature)
    np.testing.assert_allclose(got, numeric, atol=1e-8)


@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_a_tail_without_mass(temperature):
    check(*rows_without_tail_mass(), True, temperature)


@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_every_column_is_named(temperature):
    """K = cols and a teacher that sums to less than 1."""
    g = generator(302)
    z = torch.randn((3, 5), generator=g, dtype=torch.float64)
    ids = torch.stack([torch.randperm(5, generator=g) for _ in range(3)])
    teacher = torch.log_softmax(torch.randn((3, 5), generator=g, dtype=torch.float64), 1) - 0.25
    check(z, ids, teacher, True, temperature)
