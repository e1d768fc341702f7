"""A decode step's log-probabilities captured with a workspace of the size that the
library asks for (0 where rows stay whole): every replay gives the eager bits."""
import pytest
import torch

from credit_amd import hip_lib
from tests.logits_cases import make_logits
from tests.test_gpu_token_logprob import random_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols,top", [(64, 131072, 20), (1, 131072, 8), (1, 32768, 8),
                                           (300, 9001, 5)])
def test_a_captured_decode_step(gpu, rows, cols, top):
    print(f"token_logprob captured with its workspace {rows}x{cols}", flush=True)
    z = make_logits(rows, cols, "bf16", 381).to(gpu)
    tokens = random_tokens(rows, cols, 1, 382).to(gpu)
    f32 = dict(device=gpu, dtype=torch.float32)
    outs = (torch.zeros((rows, 1), **f32), torch.zeros((rows, 2), **f32), torch.zeros(rows, **f32),
            torch.zeros((rows, top), **f32), torch.zeros((rows, top), device=gpu, dtype=torch.int64))
    hip_lib.token_logprob_fwd(z, tokens, *outs)
    torch.cuda.synchronize()
    want = [t.clone() for t in outs]
    need = hip_lib.workspace_bytes("token_logprob_fwd", rows, cols)
    workspace = torch.zeros(max(need, 1), dtype=torch.uint8, device=gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cfg = hip_lib.make_cfg(workspace=workspace)
        hip_lib.token_logprob_fwd(z, tokens, *outs, 1.0, cfg)
    for i in range(5):
        for t in outs:
            t.zero_()
        graph.replay()
        hip_lib.token_logprob_fwd(z[:1], tokens[:1], *(t[:1].clone() for t in outs))
        if i % 2:
            torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i
