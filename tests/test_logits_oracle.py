"""The oracle of the operators on logits against torch in 64 bits: autograd for
the gradients, and what the definitions say of empty rows, masks and padding."""
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import reference as ref
from tests.logits_cases import generator

T = 0.7


def inputs(rows=5, cols=23, n=3):
    g = generator(3)
    z = torch.randn((rows, cols), generator=g, dtype=torch.float64) * 2
    tokens = torch.randint(0, cols, (rows, n), generator=g)
    tokens[1, 0] = -1
    tokens[2, 1] = tokens[2, 0]
    return g, z, tokens


def test_log_probabilities_and_entropy():
    _, z, tokens = inputs()
    lp = F.log_softmax(z / T, dim=1)
    logp, stats, h, top, ids = ref.token_logprob_fwd(z.numpy(), tokens.numpy(), 4, T)
    want = torch.where(tokens < 0, 0.0, lp.gather(1, tokens.clamp(min=0)))
    np.testing.assert_allclose(logp, want.numpy(), rtol=1e-12)
    np.testing.assert_allclose(h, torch.special.entr(lp.exp()).sum(1).numpy(), rtol=1e-12)
    values, columns = lp.topk(4, dim=1)
    np.testing.assert_allclose(top, values.numpy(), rtol=1e-12)
    assert np.array_equal(ids, columns.numpy())
    np.testing.assert_allclose(stats[:, 0] / T + np.log(stats[:, 1]),
                               torch.logsumexp(z / T, 1).numpy(), rtol=1e-12)


def test_order_of_equal_values_nan_and_masks():
    z = np.array([[1.0, 2.0, 2.0, -math.inf], [0.0, -0.0, 0.0, -0.0],
                  [1.0, math.nan, 5.0, math.nan], [-math.inf] * 4])
    tokens = np.array([[3], [0], [2], [1]])
    logp, stats, h, top, ids = ref.token_logprob_fwd(z, tokens, 4)
    assert ids.tolist() == [[1, 2, 0, 3], [0, 1, 2, 3], [1, 3, 2, 0], [0, 1, 2, 3]]
    assert logp[0, 0] == -math.inf and np.isnan(logp[2, 0]) and logp[3, 0] == -math.inf
    assert stats[3].tolist() == [-math.inf, 0.0] and h[3] == 0.0
    assert np.isfinite(h[0]) and (top[3] == -math.inf).all()


def test_gradient_of_log_probabilities_and_entropy():
    g, z, tokens = inputs()
    dlogp = torch.randn(tokens.shape, generator=g, dtype=torch.float64)
    dent = torch.randn(z.shape[0], generator=g, dtype=torch.float64)
    dent[3] = 0.0
    x = z.clone().requires_grad_()
    lp = F.log_softmax(x / T, dim=1)
    chosen = lp.gather(1, tokens.clamp(min=0)) * (tokens >= 0)
    ((chosen * dlogp).sum() + (torch.special.entr(lp.exp()).sum(1) * dent).sum()).backward()
    got = ref.token_logprob_bwd(z.numpy(), tokens.numpy(), dlogp.numpy(), dent.numpy(), T)
    np.testing.assert_allclose(got, x.grad.numpy(), rtol=1e-9, atol=1e-14)


@pytest.mark.parametrize("tail", [False, True])
def test_distillation_and_its_gradient(tail):
    g, z, _ = inputs()
    rows, cols = z.shape
    full = torch.randn((rows, cols), generator=g, dtype=torch.float64) * 2
    k = 6
    if tail:
        teacher, ids = F.log_softmax(full / T, dim=1).topk(k, dim=1)
    else:
        teacher, ids = full.topk(k, dim=1)
    ids[1, 2:] = -1
    ids[2] = -1
    dloss = torch.randn(rows, generator=g, dtype=torch.float64)
    x = z.clone().requires_grad_()
    p = F.softmax(x / T, dim=1)
    total = torch.zeros((), dtype=torch.float64)
    want = []
    for r in range(rows):
        live = ids[r][ids[r] >= 0]
        if live.numel() == 0:
            want.append(0.0)
            continue
        t = teacher[r][ids[r] >= 0]
        q = t.exp() if tail else F.softmax(t / T, dim=0)
        loss = (q * (q.log() - p[r, live].log())).sum()
        if tail:
            others = torch.ones(cols, dtype=torch.bool)
            others[live] = False
            rest = 1 - q.sum()
            loss = loss + rest * (rest.log() - p[r, others].sum().log())
        want.append(loss.item())
        total = total + loss * dloss[r]
    total.backward()
    got = ref.topk_distill_fwd(z.numpy(), ids.numpy(), teacher.numpy(), tail, T)
    np.testing.assert_allclose(got, want, rtol=1e-9, atol=1e-13)
    d = ref.topk_distill_bwd(z.numpy(), ids.numpy(), teacher.numpy(), dloss.numpy(), tail, T)
    np.testing.assert_allclose(d, x.grad.numpy(), rtol=1e-8, atol=1e-13)


def test_distillation_catches_a_planted_mistake():
    """A gradient that leaves out the rest's share is not the loss's."""
    g, z, _ = inputs()
    z = z[:1]
    teacher, ids = F.log_softmax(z, dim=1).topk(4, dim=1)
    z = torch.randn(z.shape, generator=g, dtype=torch.float64)
    args = (ids.numpy(), teacher.numpy())
    right = ref.topk_distill_bwd(z.numpy(), *args, np.ones(1))
    step = 1e-6
    numeric = np.array([[(ref.topk_distill_fwd(z.numpy() + step * np.eye(z.shape[1])[j], *args)
                          - ref.topk_distill_fwd(z.numpy() - step * np.eye(z.shape[1])[j], *args)
                          )[0] / (2 * step) for j in range(z.shape[1])]])
    np.testing.assert_allclose(right, numeric, atol=1e-8)
    q = np.zeros(z.shape)
    np.put_along_axis(q, ids.numpy(), np.exp(teacher.numpy()), axis=1)
    wrong = F.softmax(z, dim=1).numpy() - q
    assert np.abs(wrong - numeric).max() > 1e-3
