"""Gradients whose rows lie between the logits' own, as two column ranges of one
buffer: the bits of a gradient apart, and nothing else touched."""
import pytest
import torch

from credit_amd import hip_lib
from tests.logits_cases import DTYPES, generator, make_logits
from tests.test_gpu_token_logprob import forward, random_tokens
from tests.test_gpu_topk_distill import forward as distill
from tests.test_gpu_topk_distill import make_teacher

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [0, 1, 13])
@pytest.mark.parametrize("first", ["logits", "dlogits"])
@pytest.mark.parametrize("rows,cols", [(4, 33), (3, 8191), (5, 20003)])
def test_two_column_ranges(gpu, rows, cols, first, gap, dtype):
    print(f"gradients side by side {dtype} {rows}x{cols} {first} first, gap {gap}", flush=True)
    values = make_logits(rows, cols, dtype, 351)
    buffer = torch.full((rows, 2 * cols + 2 * gap), 3.0, dtype=DTYPES[dtype], device=gpu)
    left, right = buffer[:, :cols], buffer[:, cols + gap:2 * cols + gap]
    z, out = (left, right) if first == "logits" else (right, left)
    z.copy_(values)
    apart = torch.empty((rows, cols), dtype=DTYPES[dtype], device=gpu)
    tokens = random_tokens(rows, cols, 3, 352).to(gpu)
    dlogp = torch.randn(tokens.shape, generator=generator(353)).to(gpu)
    _, stats, _, _, _ = forward(z, tokens, 0, False)
    for d in (apart, out):
        hip_lib.token_logprob_bwd(z, tokens, stats, dlogp, d)
    torch.cuda.synchronize()
    assert torch.equal(apart, out)
    ids, teacher = make_teacher(values, 9, True, 1.0, 354)
    _, stats = distill(z, ids, teacher, True, 1.0, gpu)
    dloss = torch.ones(rows, device=gpu)
    for d in (apart, out):
        hip_lib.topk_distill_bwd(z, ids.to(gpu), teacher.to(gpu), stats, dloss, d)
    torch.cuda.synchronize()
    assert torch.equal(apart, out) and torch.equal(z.cpu(), values)
    if gap:
        assert (buffer[:, cols:cols + gap] == 3).all() and (buffer[:, -gap:] == 3).all()


def test_ranges_that_meet_are_refused(gpu):
    buffer = torch.zeros((3, 100), device=gpu)
    tokens = torch.zeros((3, 1), dtype=torch.int64, device=gpu)
    stats, dlogp = torch.ones((3, 2), device=gpu), torch.ones((3, 1), device=gpu)
    with pytest.raises(hip_lib.CreditError) as err:
        hip_lib.token_logprob_bwd(buffer[:, :50], tokens, stats, dlogp, buffer[:, 49:99])
    assert err.value.status == -8
