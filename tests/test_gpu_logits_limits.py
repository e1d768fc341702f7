"""What no rounding may break: S >= 1, for it holds its maximum's own e^0, hence
log-probabilities <= 0; entropies >= 0.  Rows whose mass lies on one token, over
many maxima."""
import math

import pytest
import torch

from credit_amd import hip_lib
from tests.logits_cases import DTYPES, generator
from tests.test_gpu_token_logprob import forward
from tests.test_gpu_topk_distill import forward as distill

pytestmark = pytest.mark.gpu


def one_token_rows(rows, cols, kind, dtype, seed):
    """Maxima spread over signs and sizes; the rest masked, far below or at a
    distance that leaves them a share of 10^-7 or so."""
    g = generator(seed)
    top = torch.randn(rows, generator=g) * torch.logspace(-2, 3, rows)
    at = torch.randint(0, cols, (rows,), generator=g)
    if kind == "masked":
        z = torch.full((rows, cols), -math.inf)
    elif kind == "lowest":
        z = torch.full((rows, cols), torch.finfo(DTYPES[dtype]).min)
    else:
        z = torch.randn((rows, cols), generator=g) + top[:, None] - 18.0 - math.log(cols)
    if kind == "late":  # first values that lie a little lower than those behind
        at = torch.full((rows,), cols - 1)
        z[:, :cols // 2] = (top - 3.0)[:, None].expand(-1, cols // 2) - 20.0
        z[:, 0] = top - 4.0
    z[torch.arange(rows), at] = top
    return z.to(DTYPES[dtype]), at[:, None]


def check(gpu, z, at, temperature, cfg, what):
    logp, stats, h, top_logp, _ = forward(z.to(gpu), at, min(z.shape[1], 3), True, temperature, cfg)
    for name, good in (("S", stats[:, 1] >= 1), ("entropy", h >= 0), ("logp", logp <= 0),
                       ("top_logp", top_logp <= 0)):
        assert good.all(), f"{what}: {(~good).sum()} rows whose {name} is beyond its limit"


@pytest.mark.parametrize("temperature", [1.0, 0.7])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["masked", "lowest", "peaked", "late"])
@pytest.mark.parametrize("cols", [1, 5, 300, 9001])
def test_one_token_holds_the_row(gpu, cols, kind, dtype, temperature):
    print(f"token_logprob limits {dtype} {cols} {kind}", flush=True)
    z, at = one_token_rows(1500, cols, kind, dtype, 341)
    check(gpu, z, at, temperature, None, kind)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["masked", "lowest", "peaked", "late"])
def test_one_token_holds_the_row_in_parts(gpu, kind, dtype):
    print(f"token_logprob limits in parts {dtype} {kind}", flush=True)
    z, at = one_token_rows(400, 25001, kind, dtype, 342)
    for parts in (2, 4):
        check(gpu, z, at, 1.0, hip_lib.make_cfg("split", parts), f"{kind} in {parts} parts")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("variant,parts", [("read", 0), ("split", 3)])
def test_sums_of_the_distillation(gpu, dtype, variant, parts):
    """S, and the tail's sum where it has mass, which one column holds here."""
    print(f"topk_distill limits {dtype} {variant}", flush=True)
    z, at = one_token_rows(400, 25001, "masked", dtype, 343)
    other = (at + 77) % 25001
    z.scatter_(1, other, 0.5 * z.gather(1, at))
    teacher = torch.full(at.shape, -0.25)
    for tail in (False, True):
        _, stats = distill(z.to(gpu), at, teacher, tail, 1.0, gpu, hip_lib.make_cfg(variant, parts))
        assert (stats[:, 1] >= 1).all()
        assert not tail or (stats[:, 3] >= 1).all()


def test_nan_and_empty_rows_stay_what_they_are(gpu):
    z = torch.full((3, 700), -math.inf)
    z[1, 5], z[2, 9] = math.nan, math.inf
    logp, stats, h, _, _ = forward(z.to(gpu), torch.full((3, 1), 5), 0)
    assert stats[0, 1] == 0 and h[0] == 0 and logp[0, 0] == -math.inf
    assert torch.isnan(stats[1:, 1]).all() and torch.isnan(h[1:]).all()
    assert torch.isnan(logp[1:]).all()
