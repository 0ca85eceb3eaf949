"""The paged step's functions as torch sees them: gradients, dispatch modes and profilers find the operators, as they
find those that are called through ``torch.ops``."""

from __future__ import annotations

import threading
import time

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from test_paged_gpu import attend, attention_problem, i32, workspace  # noqa: F401  (a fixture)

from multi_lora_b200 import paged_kv as P
from multi_lora_b200.speculative import verify_draft

pytestmark = pytest.mark.gpu


def step(dev, workspace):
    """One call of each operator: (name, call)."""
    pr = attention_problem(dev, 81, [1, 2], [20, 30], 4, 2, 64, "bf16", 16)
    plan = P.PagedStepPlan.new(2, 3, dev)
    one, free = i32([1, 1], dev), i32([4, 5], dev)
    probs, drafts = torch.full((2, 8), 0.125, device=dev), torch.zeros(1, 1, dtype=torch.long, device=dev)
    rows, u = i32([0, 2], dev), torch.zeros(1, 1, device=dev)
    head, tables, ticket, slots = (i32(x, dev) for x in ([0], [[0, -1], [1, -1]], [0], [-1] * 3))
    return [
        ("plan_paged_step", lambda: P.plan_paged_step(one, one, one, free, head, tables, plan, block_size=16,
                                                      workspace=ticket)),
        ("write_paged_kv", lambda: P.write_paged_kv(pr["q"][:, :2], pr["q"][:, 2:], pr["k"], pr["v"], slots)),
        ("paged_attention", lambda: attend(pr, workspace)),
        ("verify_draft", lambda: verify_draft(probs, None, drafts, rows, u, u[0])),
    ]


def test_dispatch_modes_see_the_operators(cuda_dev, workspace):  # noqa: F811
    seen = []

    class Names(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    for name, call in step(cuda_dev, workspace):
        plain = call()
        with Names():
            again = call()
        assert any(s.startswith(f"mlora.{name}") for s in seen), (name, seen)
        if name == "paged_attention":
            assert torch.equal(plain, again)


def test_profilers_see_the_operators(cuda_dev, workspace):  # noqa: F811
    calls = step(cuda_dev, workspace)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        for _, call in calls:
            call()
    names = {e.name for e in prof.events()}
    assert {f"mlora::{name}" for name, _ in calls} <= names


def test_a_graph_that_is_asked_for_is_not_lost_in_silence(cuda_dev, workspace):  # noqa: F811
    """There is no gradient: torch's own answer for an operator without one is what comes, not an output that
    looks like a constant."""
    pr = attention_problem(cuda_dev, 82, [1, 2], [20, 30], 4, 2, 64, "bf16", 16)
    ops = torch.ops.mlora
    with torch.no_grad():
        want = attend(dict(pr, q=pr["q"].clone().requires_grad_()), workspace)
    assert not want.requires_grad
    q = pr["q"].clone().requires_grad_()
    by_torch = ops.paged_attention(q, pr["k"], pr["v"], pr["tables"], pr["kv_lens"], pr["indptr"], 2, 64 ** -0.5, 0,
                                   None, workspace, None)
    got = attend(dict(pr, q=q), workspace)
    assert torch.equal(got, want)
    assert by_torch.requires_grad and got.requires_grad


def test_the_cache_is_no_part_of_a_graph(cuda_dev, workspace):  # noqa: F811
    """It would hold the graphs of all steps that wrote to it."""
    pr = attention_problem(cuda_dev, 83, [1, 2], [20, 30], 4, 2, 64, "bf16", 16)
    kv = pr["q"].clone().requires_grad_()
    P.write_paged_kv(kv[:, :2], kv[:, 2:], pr["k"], pr["v"], i32([0, 1, 2], cuda_dev))
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]):
        P.write_paged_kv(kv[:, :2], kv[:, 2:], pr["k"], pr["v"], i32([0, 1, 2], cuda_dev))
    assert not pr["k"].requires_grad and pr["k"].grad_fn is None and not pr["v"].requires_grad
    assert torch.equal(pr["k"][0, :3], kv[:, :2])


def test_other_threads_go_on_while_a_launch_waits(cuda_dev, workspace):  # noqa: F811
    """Behind a busy GPU the queue of launches fills up, and a launch waits for room in it."""
    _, call = step(cuda_dev, workspace)[1]
    call()
    torch.cuda.synchronize()
    gaps, stop = [], threading.Event()

    def watch():
        last = time.perf_counter()
        while not stop.is_set():
            time.sleep(0.001)
            now = time.perf_counter()
            gaps.append(now - last)
            last = now

    watcher = threading.Thread(target=watch)
    watcher.start()
    start = time.perf_counter()
    torch.cuda._sleep(1_500_000_000)  # most of a second
    for _ in range(3000):
        call()
    took = time.perf_counter() - start
    torch.cuda.synchronize()
    stop.set()
    watcher.join()
    assert took > 0.4 and max(gaps) < 0.2, (took, max(gaps))
