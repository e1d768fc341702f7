"""The gradients of normed heads, which leave partial rows between their two launches,
from one host thread while another runs other operators of the library on the same
stream: each call's bits are those it gives alone."""
import threading

import pytest
import torch

from credit_amd import hip_lib
from credit_amd.workloads import WORKLOADS
from tests.test_gpu_paged_attention import make

pytestmark = pytest.mark.gpu


def gradients(gpu, seed):
    g = torch.Generator().manual_seed(seed)
    tokens, dim = 500, 64
    xs, dys = ([torch.randn((tokens, h, dim), generator=g).to(gpu) for h in (4, 2)] for _ in "xy")
    ws = [torch.randn(dim, generator=g).to(gpu) for _ in "qk"]
    pos, freq = torch.arange(tokens, device=gpu), hip_lib.rope_frequencies(dim)[0].to(gpu)
    rstd = torch.rand((tokens, 6), generator=g).to(gpu)
    outs = [torch.empty_like(t) for t in (*xs, *ws)]
    return outs, lambda: hip_lib.qk_norm_rope_bwd(*xs, *ws, pos, freq, rstd, *dys, *outs)


def attention(gpu, seed):
    args = make([1, 1], [3000, 5000], 8, 2, 128, 16, seed=seed)
    outs = torch.empty_like(args[0]), torch.empty(args[0].shape[:2], device=gpu)
    return outs, lambda: hip_lib.paged_attention(*args, *outs)


def row_sum(gpu, seed):
    ins = tuple(t.to(gpu) for t in WORKLOADS["row_sum_max"].make_inputs(4, 300000, seed=seed))
    outs = hip_lib.allocate_outputs("row_sum_max", ins)
    return outs, lambda: hip_lib.HIP_LAUNCHERS["row_sum_max"](ins, outs)


@pytest.mark.parametrize("other", [gradients, attention, row_sum])
def test_two_threads_on_one_stream(gpu, other):
    print(f"gradients beside {other.__name__}", flush=True)
    cases = [gradients(gpu, 1), other(gpu, 2)]
    alone = []
    for outs, call in cases:
        call()
        torch.cuda.synchronize()
        alone.append([t.clone() for t in outs])
    stream = torch.cuda.Stream()
    for outs, call in cases:  # the workspace of the stream is there
        with torch.cuda.stream(stream):
            call()
    torch.cuda.synchronize()
    start, done, errors = threading.Barrier(4), threading.Event(), []

    def beside(call):
        try:
            with torch.cuda.stream(stream):
                start.wait(timeout=30)
                for _ in range(20000):
                    if done.is_set():
                        break
                    call()
        except Exception as e:  # noqa: BLE001 (reported by the test's thread)
            errors.append(repr(e))

    threads = [threading.Thread(target=beside, args=(cases[1][1],)) for _ in range(3)]
    for t in threads:
        t.start()
    outs, call = cases[0]
    wrong = torch.zeros((), dtype=torch.int64, device=gpu)
    with torch.cuda.stream(stream):
        start.wait(timeout=30)
        for _ in range(1000):
            call()
            for t, e in zip(outs, alone[0]):
                wrong += (t != e).sum()
    done.set()
    for t in threads:
        t.join(timeout=60)
    torch.cuda.synchronize()
    assert int(wrong) == 0
    assert not errors and not any(t.is_alive() for t in threads), errors
    # The other's last calls, too.
    assert all(torch.equal(a, b) for a, b in zip(cases[1][0], alone[1]))
