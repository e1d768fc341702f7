"""Rows of the logits forwards in several parts (SPLIT, and AUTO for few rows):
against the oracle, repeatedly on one workspace, from two threads, under capture
and beside each other."""
import threading

import pytest
import torch

from credit_amd import hip_lib
from tests.logits_cases import DTYPES, make_logits, placed, special_rows
from tests.test_gpu_token_logprob import check_forward, random_tokens
from tests.test_gpu_token_logprob import forward as logprob
from tests.test_gpu_topk_distill import check_loss, make_teacher
from tests.test_gpu_topk_distill import forward as distill

pytestmark = pytest.mark.gpu

SHAPES = [(1, 8193), (3, 16384), (5, 50001), (2, 131072), (1, 300007), (2, 1100001)]


def split(p, workspace=None):
    return hip_lib.make_cfg("split", p, workspace=workspace)


@pytest.mark.parametrize("parts", [0, 2, 3, 7, 64])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forwards_in_parts(gpu, rows, cols, dtype, parts):
    print(f"logits split {parts} {dtype} {rows}x{cols}", flush=True)
    z = make_logits(rows, cols, dtype, 81)
    zs = placed(z, gpu, 1, 2) if parts == 3 else z.to(gpu)
    tokens = random_tokens(rows, cols, 3, 82)
    check_forward(z, tokens, 33, logprob(zs, tokens, 33, cfg=split(parts)))
    check_forward(z, tokens, 0, logprob(zs, tokens, 0, False, cfg=split(parts)))
    for tail in (False, True):
        ids, teacher = make_teacher(z, 40, tail, 1.0, 83)
        if tail:
            ids[0, 7], teacher[0] = ids[0, 3], teacher[0] - 1.0  # one column twice
            ids[-1, 5:] = -1
        loss, _ = distill(zs, ids, teacher, tail, 1.0, gpu, split(parts))
        check_loss(z, ids, teacher, tail, 1.0, loss)


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_rows_in_parts(gpu, dtype):
    cols = 40003
    print(f"logits split special rows {dtype}", flush=True)
    z, names = special_rows(cols, dtype, 84)
    tokens = torch.tensor([[0, cols // 2, cols - 1, -1, cols]] * len(names))
    got = logprob(z.to(gpu), tokens, 40, cfg=split(4))
    losses = []
    for tail in (False, True):
        ids, teacher = make_teacher(z, 9, tail, 1.0, 85)
        ids[0] = -1
        losses.append((tail, ids, teacher, distill(z.to(gpu), ids, teacher, tail, 1.0, gpu,
                                                   split(4))[0]))
    for i, name in enumerate(names):
        s = slice(i, i + 1)
        check_forward(z[s], tokens[s], 40, [t[s] for t in got], 1.0, name)
        for tail, ids, teacher, loss in losses:
            check_loss(z[s], ids[s], teacher[s], tail, 1.0, loss[s], name)


def call_of(gpu, seed, rows=6, cols=131072, cfg=None, dtype="bf16"):
    """(outputs, call) of a forward with alternatives and one with a tail."""
    z = make_logits(rows, cols, dtype, seed).to(gpu)
    tokens = random_tokens(rows, cols, 2, seed).to(gpu)
    ids, teacher = (t.to(gpu) for t in make_teacher(z.cpu(), 16, True, 1.0, seed))
    f32 = dict(device=gpu, dtype=torch.float32)
    outs = (torch.zeros((rows, 2), **f32), torch.zeros((rows, 2), **f32),
            torch.zeros(rows, **f32), torch.zeros((rows, 9), **f32),
            torch.zeros((rows, 9), device=gpu, dtype=torch.int64), torch.zeros(rows, **f32),
            torch.zeros((rows, 8), **f32))

    def call():
        hip_lib.token_logprob_fwd(z, tokens, *outs[:5], cfg=cfg)
        hip_lib.topk_distill_fwd(z, ids, teacher, *outs[5:], cfg=cfg)
    return outs, call


def clear(outs):
    for t in outs:
        t.zero_()


def test_one_workspace_again_and_again(gpu):
    """Counters are 0 again after every call, whatever the shapes: 40 calls give
    the bits of the first; a workspace that is too small is refused."""
    print("logits split repeated", flush=True)
    need = max(hip_lib.workspace_bytes("token_logprob_fwd", r, 131072, "split", p)
               for r, p in ((6, 16), (200, 3)))
    ws = torch.zeros(need, dtype=torch.uint8, device=gpu)
    calls = [call_of(gpu, 86, cfg=split(16, ws)), call_of(gpu, 87, 200, 20003, split(3, ws)),
             call_of(gpu, 88, 3, 131072, split(5, ws), "f32")]
    firsts = []
    for outs, call in calls:
        call()
        torch.cuda.synchronize()
        firsts.append([t.clone() for t in outs])
    for i in range(40):
        outs, call = calls[i % 3]
        clear(outs)
        call()
        assert all(torch.equal(a, b) for a, b in zip(outs, firsts[i % 3]))
    assert not ws[256:256 + (1 << 20)].any()
    _, call = call_of(gpu, 86, cfg=split(16, ws[:(5 << 20) + 1024]))
    with pytest.raises(hip_lib.CreditError) as err:
        call()
    assert err.value.status == -5


@pytest.mark.parametrize("streams", [1, 2])
def test_two_threads(gpu, streams):
    print(f"logits split two threads on {streams} stream(s)", flush=True)
    cases = [call_of(gpu, 89), call_of(gpu, 90, 3, 262144)]
    alone = []
    for outs, call in cases:
        call()
        torch.cuda.synchronize()
        alone.append([t.clone() for t in outs])
    shared = [torch.cuda.Stream() for _ in range(streams)]
    torch.cuda.synchronize()
    start, errors = threading.Barrier(2), []

    def work(i):
        outs, call = cases[i]
        wrong = torch.zeros((), dtype=torch.int64, device=gpu)
        try:
            with torch.cuda.stream(shared[i % streams]):
                start.wait(timeout=30)
                for _ in range(50):
                    clear(outs)
                    call()
                    for t, e in zip(outs, alone[i]):
                        wrong += (t != e).sum()
            shared[i % streams].synchronize()
            if int(wrong):
                errors.append((i, int(wrong)))
        except Exception as e:  # noqa: BLE001 (reported by the test's thread)
            errors.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=60)
    assert not errors and not any(t.is_alive() for t in threads), errors


def capture(call):
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    return graph


def test_capture(gpu):
    """A captured call has a workspace of its own, or none (one workgroup a row,
    the values within rounding); replays beside eager calls and each other."""
    print("logits under capture", flush=True)
    rows, cols = 6, 131072
    need = hip_lib.workspace_bytes("token_logprob_fwd", rows, cols)
    graphs = []
    for seed in (91, 92):
        ws = torch.zeros(need, dtype=torch.uint8, device=gpu)
        cfg = hip_lib.make_cfg(workspace=ws)
        outs, call = call_of(gpu, seed, cfg=cfg)
        call()
        torch.cuda.synchronize()
        want = [t.clone() for t in outs]

        def captured(outs=outs, call=call, cfg=cfg):
            cfg.stream = torch.cuda.current_stream().cuda_stream
            call()
        graphs.append((capture(captured), outs, want, ws, cfg, call))
    # No workspace: one workgroup a row.
    outs, call = call_of(gpu, 93)
    call()
    torch.cuda.synchronize()
    plain = [t.clone() for t in outs]
    graph = capture(call)
    eager, eager_call = call_of(gpu, 94)
    eager_call()
    torch.cuda.synchronize()
    first = [t.clone() for t in eager]
    streams = [torch.cuda.Stream() for _ in range(3)]
    for i in range(6):
        for t in [*eager, *outs, *graphs[0][1], *graphs[1][1]]:
            t.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, (graph, graphs[0][0], graphs[1][0])):
            with torch.cuda.stream(s):
                g.replay()
        eager_call()
        if i % 2:
            torch.cuda.synchronize()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, first))
        for _, got, want, *_ in graphs:
            assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        for a, b in zip(outs, plain):
            assert torch.allclose(a.double(), b.double(), rtol=1e-5, atol=1e-5), i


def test_split_under_capture_needs_a_workspace(gpu):
    print("logits SPLIT under capture without a workspace", flush=True)
    z = make_logits(2, 131072, "bf16", 95).to(gpu)
    tokens = torch.zeros((2, 1), dtype=torch.int64, device=gpu)
    logp, stats = torch.zeros((2, 1), device=gpu), torch.zeros((2, 2), device=gpu)
    seen = []

    def call():
        logp.add_(1.0)
        try:
            hip_lib.token_logprob_fwd(z, tokens, logp, stats, cfg=split(4))
        except hip_lib.CreditError as e:
            seen.append(e.status)
    graph = capture(call)
    graph.replay()
    torch.cuda.synchronize()
    assert seen == [-5] and (logp == 1.0).all()


def test_another_stream_and_its_own_rows(gpu):
    """A call on a stream of its own that its caller waits for; the tensors were
    made on another."""
    print("logits on another stream", flush=True)
    outs, call = call_of(gpu, 96)
    call()
    torch.cuda.synchronize()
    want = [t.clone() for t in outs]
    stream = torch.cuda.Stream()
    for _ in range(3):
        clear(outs)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            call()
        torch.cuda.current_stream().wait_stream(stream)
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, want))

