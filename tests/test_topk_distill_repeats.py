"""The oracle's distillation where entries name one column more than once: the KL
of their sum, against the definition over dense rows."""
import math

import numpy as np
import pytest
import torch

from oracle import reference as ref
from tests import distill_definition as definition
from tests.logits_cases import generator


def test_equal_entries_of_one_column():
    """Two entries of one column are one of twice the mass."""
    z = np.array([[0.0, 5.0, 0.0, 0.0]])
    once = ref.topk_distill_fwd(z, [[1]], np.array([[0.0]]), False)
    twice = ref.topk_distill_fwd(z, [[1, 1]], np.array([[3.0, 3.0]]), False)
    np.testing.assert_allclose(twice, once, rtol=1e-14)
    assert twice[0] > 0.0
    q = np.log([[0.5, 0.25]])
    np.testing.assert_allclose(ref.topk_distill_fwd(z, [[1, 1]], q, True),
                               ref.topk_distill_fwd(z, [[1]], np.log([[0.75]]), True), rtol=1e-14)


@pytest.mark.parametrize("tail", [False, True])
def test_repeats_among_others(tail):
    g = generator(321)
    z = torch.randn((5, 19), generator=g, dtype=torch.float64)
    ids = torch.randint(0, 19, (5, 12), generator=g)
    ids[0, ::3] = -1
    ids[1] = 7
    ids[2, 1:5] = ids[2, 0]
    teacher = torch.randn((5, 12), generator=g, dtype=torch.float64)
    if tail:
        teacher = torch.log_softmax(teacher, 1) - 0.25
    teacher[2, 2] = -math.inf
    teacher[3, 4:] = -math.inf
    ids[3, 5] = ids[3, 4]
    args = (ids.numpy(), teacher.numpy())
    got = ref.topk_distill_fwd(z.numpy(), *args, tail, 0.7)
    want = definition.loss(z, ids, teacher, tail, 0.7).numpy()
    np.testing.assert_allclose(got, want, rtol=1e-12)
    # Twice the same student and teacher: a KL is at least 0.
    assert tail or (got >= 0).all()
    dloss = torch.ones(5, dtype=torch.float64)
    np.testing.assert_allclose(ref.topk_distill_bwd(z.numpy(), *args, np.ones(5), tail, 0.7),
                               definition.gradient(z, ids, teacher, dloss, tail, 0.7).numpy(),
                               atol=1e-13)
