"""The plans of a PagedKVCache: one for each size, at the same addresses for as long as the cache lives (no GPU needed)."""

from __future__ import annotations

import gc
import weakref

import torch

from multi_lora_b200 import paged_kv as P


def addresses(plan):
    return [t.data_ptr() for t in (plan.q_indptr, plan.kv_lens, plan.held_blocks, plan.free_head, plan.positions,
                                   plan.slot_map)]


def test_a_plan_outlives_steps_of_other_sizes(monkeypatch):
    """A captured graph has the addresses of its step's plan and nothing else that holds it."""
    planned = []
    monkeypatch.setattr(P, "plan_paged_step", lambda *a, **k: planned.append(a[6]) or a[6])
    cache = P.PagedKVCache(layers=1, num_blocks=4, block_size=4, kv_heads=1, head_dim=8, max_requests=2, max_blocks=2,
                           dtype=torch.float32, device=torch.device("cpu"))
    new = torch.zeros(2, dtype=torch.int32)
    cache.plan(new, 8)
    alive = [weakref.ref(t) for t in (cache.plan_now.q_indptr, cache.plan_now.kv_lens, cache.plan_now.positions,
                                      cache.plan_now.slot_map)]
    at = addresses(cache.plan_now)
    for size in (300, 8, 17, 300, 64):
        cache.plan(new, size)
        planned.clear()
        gc.collect()
        assert all(ref() is not None for ref in alive)
        assert cache.plan_now.slot_map.numel() == cache.plan_now.positions.numel() == size
        assert cache.plan_now.held_blocks is cache.held_blocks and cache.plan_now.free_head is cache.free_head
    assert addresses(cache.plan(new, 8)) == at
    assert addresses(cache.plan(new, 300)) != at and cache.plan_now.slot_map.numel() == 300
