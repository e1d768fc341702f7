"""The gradients on logits within bounds that follow each element's own
exponent and terms (tests/logits_bounds.py): some 10^-6 of p, and of a teacher's q
by itself."""
import numpy as np
import pytest
import torch

from credit_amd import hip_lib
from oracle import reference as ref
from tests import distill_definition as definition
from tests.logits_bounds import (ONE_BATCH, distill_gradient_bound, logprob_gradient_bound,
                                 rounded)
from tests.logits_cases import DTYPES, as64, assert_within, generator, make_logits
from tests.test_gpu_token_logprob import backward as logprob_backward
from tests.test_gpu_token_logprob import random_tokens
from tests.test_gpu_topk_distill import backward as distill_backward
from tests.test_gpu_topk_distill import make_teacher
from tests.test_logits_bounds import far_teacher

pytestmark = pytest.mark.gpu

COLS = [1, 40, 257, 4099, ONE_BATCH]


@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 0.75, 2.0])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS)
def test_log_probability_gradients(gpu, cols, dtype, temperature, entropy):
    print(f"token_logprob_bwd bounds {dtype} {cols} T {temperature}", flush=True)
    rows = 24
    z = make_logits(rows, cols, dtype, 361)
    z[1] *= 4.0
    z[2, ::2] = -torch.inf if cols > 1 else z[2, 0]
    tokens = random_tokens(rows, cols, 2, 362)
    dlogp = torch.randn(tokens.shape, generator=generator(363))
    dent = torch.randn(rows, generator=generator(364)) if entropy else None
    out = logprob_backward(z.to(gpu), tokens, dlogp, dent, temperature, gpu)
    dent64 = None if dent is None else as64(dent)
    want = ref.token_logprob_bwd(as64(z), tokens.numpy(), as64(dlogp), dent64, temperature)
    bound = logprob_gradient_bound(as64(z), tokens.numpy(), as64(dlogp), dent64, temperature)
    assert_within(as64(out), want, rounded(bound, want, z.dtype), "dlogits")


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 0.75, 2.0])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS)
def test_distillation_gradients(gpu, cols, dtype, temperature, tail):
    print(f"topk_distill_bwd bounds {dtype} {cols} T {temperature} tail {tail}", flush=True)
    rows = 24
    z = make_logits(rows, cols, dtype, 365)
    z[1] *= 4.0
    ids, teacher = make_teacher(z, 16, tail, temperature, 366)
    ids[3, 5:] = -1
    ids[4, 1] = ids[4, 0]
    if tail:
        teacher[4] -= 1.0
    dloss = torch.randn(rows, generator=generator(367))
    out = distill_backward(z.to(gpu), ids, teacher, dloss, tail, temperature, gpu)
    want = definition.gradient(z, ids, teacher, dloss, tail, temperature).numpy()
    bound = distill_gradient_bound(as64(z), ids, as64(teacher), as64(dloss), tail, temperature)
    assert_within(as64(out), want, rounded(bound, want, z.dtype), "dlogits")


@pytest.mark.parametrize("cols", [300, 5003])
def test_teachers_far_from_0(gpu, cols):
    """Logits near 24 at T = 0.7: a log-sum of 34 rounded to fp32 is off by 2e-6."""
    print(f"topk_distill_bwd teacher far from 0, {cols}", flush=True)
    z, ids, teacher, temperature = far_teacher(cols)
    dloss = torch.ones(len(z))
    out = distill_backward(z.to(gpu), ids, teacher, dloss, False, temperature, gpu)
    want = definition.gradient(z, ids, teacher, dloss, False, temperature).numpy()
    bound = distill_gradient_bound(as64(z), ids, as64(teacher), as64(dloss), False, temperature)
    assert_within(as64(out), want, bound, "dlogits")
    at = ids.numpy()
    assert (np.take_along_axis(bound, at, 1) < 2e-6 * -np.take_along_axis(want, at, 1)).mean() > 0.9
