"""Calls of the operators of a served layer that its programs make around their ordinary ones: several threads, and what a call refuses."""
import threading

import pytest
import torch

from jarvis_b200 import _lib, ops
from tests import test_gpu_gated_delta as delta

pytestmark = pytest.mark.gpu
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def test_two_threads_on_one_stream():
    """Prompts in segments, whose calls launch three kernels around scratch of their own: the bits of calls alone."""
    B, T, H = 1, 2500, 4
    problems = [delta._problem(B, T, H, H, seed=s) for s in (21, 22)]
    assert _lib.load().jb200_gated_delta_scratch_bytes(B, T, H) > 0

    def work(p):
        return ops.gated_delta_scan(*p[:5], B, T, H, state_in=p[5], want_state=True)

    alone = [work(p) for p in problems]
    torch.cuda.synchronize()
    results, start = [[], []], threading.Barrier(2)

    def run(i):
        start.wait()
        for _ in range(40):
            results[i].append(work(problems[i]))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for got, want in zip(results, alone):
        assert len(got) == 40 and all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("T", [1, 9, 200, 1500])
def test_gates_with_row_strides_of_their_own(T):
    """A slice of one projection beside a tensor of its own: the bits of two contiguous ones."""
    B, H = 1, 3
    q, k, v, g, b, s = delta._problem(B, T, H, H, seed=31)
    wide = torch.full((B * T, 2 * H + 1), float("nan"), device="cuda")
    wide[:, :H], wide[:, H:2 * H] = g, b
    want = ops.gated_delta_scan(q, k, v, g, b, B, T, H, state_in=s, want_state=True)
    for log_decay, beta in ((wide[:, :H], b), (g, wide[:, H:2 * H]), (wide[:, :H], wide[:, H:2 * H])):
        got = ops.gated_delta_scan(q, k, v, log_decay, beta, B, T, H, state_in=s, want_state=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
