"""Requests without new tokens: a cache plans all requests that it has room for at every step, and most may be idle."""

from __future__ import annotations

import pytest
import torch

from test_paged_gpu import assert_attention, attend, attention_problem, status_word, workspace  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def spread(requests, active):
    """q_lens of a few active requests among many."""
    lens = [0] * requests
    for i, q in active.items():
        lens[i] = q
    return lens


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("requests, active, heads", [
    (40, {0: 1, 39: 2}, (8, 2)),                                     # decode kernel
    (1500, {0: 1, 31: 1, 32: 2, 33: 1, 64: 2, 500: 1, 1499: 2}, (8, 2)),
    (700, {i: 1 for i in range(3, 700, 41)}, (8, 8)),
    (600, {288: 1, 289: 1, 545: 1, 546: 1}, (8, 2)),                 # 256 idle ones between, from a request's 33rd on
    (300, {0: 30, 150: 200, 299: 5}, (8, 2)),                        # chunk kernel
    (1200, {i: 1 + i % 70 for i in range(0, 1200, 97)}, (8, 2)),
])
def test_few_active_among_many(cuda_dev, workspace, requests, active, heads, dtype):  # noqa: F811
    q_lens = spread(requests, active)
    kv_lens = [q + 37 * i % 900 if q else 5 * (i % 3) for i, q in enumerate(q_lens)]
    pr = attention_problem(cuda_dev, 91, q_lens, kv_lens, *heads, 64, dtype, 16, spare_rows=2)
    status = status_word(cuda_dev)
    got = attend(pr, workspace, status=status)
    assert status.item() == 0
    assert (got[sum(q_lens):] == 0).all()
    assert_attention(got, pr, dtype)


def device_us(call, n=20):
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(n):
            call()
    times = []
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3 / n)
    return min(times)


@pytest.mark.parametrize("q", [1, 64])
def test_idle_requests_cost_next_to_nothing(cuda_dev, workspace, q):  # noqa: F811
    """Two active requests at the ends of a thousand: one at a time, the idle ones between them took 20 times as long
    as the two alone; twice as long is allowed."""
    times = []
    for requests in (2, 1024):
        lens = spread(requests, {0: q, requests - 1: q})
        pr = attention_problem(cuda_dev, 92, lens, [3000 if n else 0 for n in lens], 32, 8, 128, "bf16", 16)
        out = torch.empty_like(pr["q"])
        times.append(device_us(lambda: attend(pr, workspace, out=out)))
    assert times[1] < 2 * times[0] + 5, times
