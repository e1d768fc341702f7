"""The operators on logits as a training and a serving program use them
together: a teacher's pass keeps its alternatives, a student learns from them and
from a policy loss with an entropy bonus, all captured into a graph too."""
import numpy as np
import pytest
import torch

from credit_amd import hip_lib
from oracle import reference as ref
from tests.logits_cases import DTYPES, as64, generator, half_step, make_logits, sum_error

pytestmark = pytest.mark.gpu


class Step:
    """Gradient of sum(w kl) + sum(a logp) + sum(b entropy) for a student's
    logits; the teacher's entries come from its own logits."""

    def __init__(self, gpu, dtype, rows, cols, k, temperature, seed):
        g = generator(seed)
        self.temperature = temperature
        self.teacher_z = make_logits(rows, cols, dtype, seed)
        noise = torch.randn((rows, cols), generator=g)
        self.z = (self.teacher_z.float() + noise).to(DTYPES[dtype])
        self.tokens = torch.randint(0, cols, (rows, 1), generator=g)
        self.tokens[-1] = -1
        self.w, self.a, self.b = (torch.randn(rows, generator=g) for _ in range(3))
        self.b[-1] = 0.0
        f32 = dict(device=gpu, dtype=torch.float32)
        dev = lambda t: t.to(gpu)  # noqa: E731
        self.g = {n: dev(getattr(self, n)) for n in ("teacher_z", "z", "tokens", "w", "b")}
        self.g["a"] = dev(self.a)[:, None].contiguous()
        self.none = torch.zeros((rows, 0), device=gpu, dtype=torch.int64)
        self.no_logp = torch.zeros((rows, 0), **f32)
        self.top_logp = torch.zeros((rows, k), **f32)
        self.top_ids = torch.zeros((rows, k), device=gpu, dtype=torch.int64)
        self.logp, self.loss, self.entropy = (torch.zeros(s, **f32)
                                              for s in ((rows, 1), (rows,), (rows,)))
        self.stats, self.stats8 = torch.zeros((rows, 2), **f32), torch.zeros((rows, 8), **f32)
        self.d_kl = torch.zeros_like(self.g["z"])
        self.d_policy = torch.zeros_like(self.g["z"])

    def __call__(self):
        g, t = self.g, self.temperature
        hip_lib.token_logprob_fwd(g["teacher_z"], self.none, self.no_logp, self.stats,
                                  top_logp=self.top_logp, top_ids=self.top_ids, temperature=t)
        hip_lib.topk_distill_fwd(g["z"], self.top_ids, self.top_logp, self.loss, self.stats8,
                                 temperature=t)
        hip_lib.topk_distill_bwd(g["z"], self.top_ids, self.top_logp, self.stats8, g["w"],
                                 self.d_kl, temperature=t)
        hip_lib.token_logprob_fwd(g["z"], g["tokens"], self.logp, self.stats, self.entropy)
        hip_lib.token_logprob_bwd(g["z"], g["tokens"], self.stats, g["a"], self.d_policy,
                                  self.entropy, g["b"])

    def outputs(self):
        return (self.top_logp, self.top_ids, self.loss, self.d_kl, self.logp, self.entropy,
                self.d_policy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(5, 4099), (3, 131072), (40, 20003)])
def test_a_training_step(gpu, rows, cols, dtype):
    print(f"logits step {dtype} {rows}x{cols}", flush=True)
    k, temperature = 24, 2.0
    step = Step(gpu, dtype, rows, cols, k, temperature, 101)
    step()
    torch.cuda.synchronize()
    _, _, _, top, ids = ref.token_logprob_fwd(as64(step.teacher_z), step.tokens.numpy(), k,
                                              temperature)
    assert np.array_equal(step.top_ids.cpu().numpy(), ids)
    # The loss of the exact teacher: its log-probabilities are off by ln S's error
    # and a rounding, the student's ln p by its own; all weighed by q.
    err = sum_error(cols)
    loss = ref.topk_distill_fwd(as64(step.z), ids, top, True, temperature)
    bound = 4 * (err + np.abs(top).max() * 2.0 ** -24) * (1 + np.abs(loss)) + 1e-7
    assert (np.abs(as64(step.loss) - loss) <= bound).all()
    d = ref.topk_distill_bwd(as64(step.z), ids, top, as64(step.w), True, temperature)
    p = np.exp(ref._log_softmax(as64(step.z), temperature)[2])
    w = np.abs(as64(step.w))[:, None] / temperature
    bound = (w * (4 * p + np.abs(d) / w) * (1.7e-5 + 6 * err) + 1e-30
             + np.abs(d) * half_step(dtype) * (1 + 1e-6))
    assert (np.abs(as64(step.d_kl) - d) <= bound).all()
    # The policy part by the chain rule in 64 bits.
    x = step.z.double().requires_grad_()
    lp = torch.log_softmax(x, 1)
    chosen = lp.gather(1, step.tokens.clamp(min=0))[:, 0] * (step.tokens[:, 0] >= 0)
    entropy = torch.special.entr(lp.exp()).sum(1)
    ((chosen * step.a).sum() + (entropy * step.b).sum()).backward()
    want = x.grad.numpy()
    p = lp.exp().detach().numpy()
    weight = (np.abs(as64(step.a)) + np.abs(as64(step.b)) * 40)[:, None]
    bound = (p * weight + np.abs(want)) * (1.7e-5 + 3 * err) + 1e-7 * weight * p + 1e-30
    bound = bound + np.abs(want) * half_step(dtype) * (1 + 1e-6)
    assert (np.abs(as64(step.d_policy) - want) <= bound).all()
    assert (step.d_policy[-1] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_captured_step(gpu, dtype):
    """Replayed several times with eager work between: every replay's gradients
    are the eager step's (rows enough that no workspace is used)."""
    print(f"logits step captured {dtype}", flush=True)
    step = Step(gpu, dtype, 300, 20003, 16, 1.0, 102)
    step()
    torch.cuda.synchronize()
    want = [t.clone() for t in step.outputs()]
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    other = Step(gpu, dtype, 300, 20003, 16, 1.0, 103)
    for i in range(5):
        for t in step.outputs():
            t.zero_()
        graph.replay()
        other()
        if i % 2:
            torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(step.outputs(), want)), i
