"""A paged KV cache: block tables and slots of a step, the cache write, and attention over it.

The reference keeps one dense row of ``max_len`` positions per request in the
model library's cache. Here keys and values live in blocks of ``block_size``
slots that requests take from a common free list as they grow; every length,
table and free list stays on the GPU, so a step needs no host round trip and
may be captured in a CUDA graph:

    plan_paged_step   lengths -> blocks, slots, positions, q_indptr
    write_paged_kv    new keys and values into their slots
    paged_attention   the new tokens' queries over the cache

``q_indptr`` has the layout of ``KernelInputMetaData.seg_indptr`` with one
segment a request, so the LoRA projections of the step can be routed by it.
:class:`PagedKVCache` holds the state between steps.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence

import torch

from multi_lora_b200 import _native

# what paged_attention asks of a workspace, whatever the shapes (mlora_paged_attention_workspace_bytes)
ATTENTION_WORKSPACE_BYTES = 64 << 20

_STATUS_TEXT = {
    0x4: "q_indptr or row_indptr decreasing or past the row count",
    0x10: "an asynchronous copy did not complete in time",
    0x20: "a length or count is negative or past its table or buffer",
    0x40: "the free list ended before every request had its blocks",
    0x80: "a slot or block-table entry outside the cache",
    0x100: "a drafted token outside the vocabulary",
}


def _need_cuda(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"mlora: {what} needs CUDA tensors (no CPU path)")


def check_status(status: torch.Tensor) -> None:
    """Raise if a launch that was given ``status`` met invalid lengths, tables or
    tokens (synchronises); the word is cleared."""
    bits = int(status.item())
    if bits:
        status.zero_()
        raise RuntimeError("mlora: invalid paged step: " + "; ".join(t for b, t in _STATUS_TEXT.items() if bits & b))


def attention_workspace(device: torch.device) -> torch.Tensor:
    """A workspace for :func:`paged_attention`; calls that may overlap on the GPU need one each. Its
    first 4 KiB are counters, zero between calls; they are to be zeroed again after a call that reported a
    copy that did not complete in time."""
    return torch.zeros(ATTENTION_WORKSPACE_BYTES, dtype=torch.uint8, device=device)


@dataclass
class PagedStepPlan:
    """What :func:`plan_paged_step` writes; int32 CUDA tensors whose addresses stay fixed from step to step."""

    q_indptr: torch.Tensor     # [R + 1] first token of each request
    kv_lens: torch.Tensor      # [R] tokens in the cache with the step's own
    held_blocks: torch.Tensor  # [R] entries of its table row that a request holds now
    free_head: torch.Tensor    # [1] first free entry of the free list now
    positions: torch.Tensor    # [max_tokens] position of each token in its request
    slot_map: torch.Tensor     # [max_tokens] block * block_size + offset, -1 without a block

    @classmethod
    def new(cls, requests: int, max_tokens: int, device: torch.device) -> "PagedStepPlan":
        def i32(n):
            return torch.zeros(n, dtype=torch.int32, device=device)

        return cls(i32(requests + 1), i32(requests), i32(requests), i32(1), i32(max_tokens), i32(max_tokens))


def plan_paged_step(ctx_lens: torch.Tensor, new_lens: torch.Tensor, held_blocks: torch.Tensor,
                    free_blocks: torch.Tensor, free_head: torch.Tensor, block_tables: torch.Tensor,
                    plan: PagedStepPlan, *, block_size: int, workspace: torch.Tensor,
                    status: Optional[torch.Tensor] = None) -> PagedStepPlan:
    """Blocks, slots, positions and offsets of a step in one launch; all int32 on one device.

    Request i (``ctx_lens[i]`` tokens in the cache, ``new_lens[i]`` more) takes
    the blocks that it lacks from ``free_blocks[free_head:]``, requests in
    order, and they are written into its row of ``block_tables`` behind the
    ``held_blocks[i]`` it has. Where the free list ends, the tokens left over get
    slot -1 (and ``status`` is marked). ``plan.held_blocks`` / ``plan.free_head``
    may be ``held_blocks`` / ``free_head`` themselves; without that, planning
    again from the same inputs writes the same plan. ``workspace``: int32 [1],
    zero before its first use, not shared by calls that overlap on the GPU.
    """
    _need_cuda(ctx_lens, "plan_paged_step")
    _native.direct("plan_paged_step")(ctx_lens, new_lens, held_blocks, free_blocks, free_head, block_tables, block_size,
                                  plan.q_indptr, plan.kv_lens, plan.held_blocks, plan.free_head, plan.positions,
                                  plan.slot_map, workspace, status)
    return plan


def write_paged_kv(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   slot_map: torch.Tensor, *, status: Optional[torch.Tensor] = None) -> None:
    """``cache[slot // block_size, slot % block_size] = k[t], v[t]`` for every slot >= 0, in place.

    k, v [tokens, kv_heads, head_dim] (slices of a fused q/k/v output are read
    where they are), caches [num_blocks, block_size, kv_heads, head_dim] of any
    strides with head_dim innermost, slot_map int32 [tokens] without repeats.
    """
    _need_cuda(k, "write_paged_kv")
    _native.direct("write_paged_kv")(k, v, k_cache, v_cache, slot_map, status)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                    kv_lens: torch.Tensor, q_indptr: torch.Tensor, *, max_q_len: int, workspace: torch.Tensor,
                    scale: Optional[float] = None, window: int = 0, out: Optional[torch.Tensor] = None,
                    status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of each request's new tokens over its cached keys (its own new ones among them).

    q [tokens, q_heads, head_dim]: request i's are rows q_indptr[i] ..
    q_indptr[i+1] - 1, the last of them at position kv_lens[i] - 1. Query head h
    reads key head h // (q_heads // kv_heads). ``window`` > 0 limits a query to
    that many keys, its own among them. ``max_q_len``: the longest request's
    new tokens, or more, on the host. The width of ``block_tables`` bounds the keys: a
    view of its first columns lets a few short requests take a launch of lower
    latency. ``workspace``: :func:`attention_workspace`.
    Queries that see no key and rows past q_indptr[-1] give zeros; rows of a request with more new tokens than
    ``max_q_len`` or with offsets that make no sense are reported in ``status`` and are zeros where they are not
    computed. What a query does not see does not reach it, infinities and NaN included. bfloat16,
    float16 or float32; head_dim a multiple of 8, at most 256; the tensor-core
    kernels take 16-bit caches with head_dim up to 128 and blocks of a multiple of 8 slots.
    """
    _need_cuda(q, "paged_attention")
    if scale is None:
        scale = q.shape[-1] ** -0.5
    return _native.direct("paged_attention")(q, k_cache, v_cache, block_tables, kv_lens, q_indptr, max_q_len, scale, window,
                                         out, workspace, status)


class PagedKVCache:
    """The state of a paged cache between steps: blocks, tables, lengths and the free list, for ``layers`` layers.

        cache.plan(new_lens, max_tokens)        # once a step
        cache.write(layer, k, v)                # per layer
        o = cache.attend(layer, q, max_q_len)
        cache.advance(num_new)                  # tokens that stay (all of them, or those that verification kept)

    Blocks are stored head by head ([num_blocks, kv_heads, block_size, head_dim]),
    so that what one head's attention reads of a block is one piece of memory.
    """

    def __init__(self, *, layers: int, num_blocks: int, block_size: int, kv_heads: int, head_dim: int,
                 max_requests: int, max_blocks: int, dtype: torch.dtype, device: torch.device) -> None:
        if min(layers, num_blocks, block_size, kv_heads, head_dim, max_requests, max_blocks) < 1:
            raise ValueError("PagedKVCache: every size must be positive")
        shape = (layers, 2, num_blocks, kv_heads, block_size, head_dim)
        self.storage = torch.zeros(shape, dtype=dtype, device=device)
        self.block_size, self.num_blocks, self.device = block_size, num_blocks, torch.device(device)

        def i32(*shape, value=0):
            return torch.full(shape, value, dtype=torch.int32, device=device)

        self.block_tables = i32(max_requests, max_blocks, value=-1)
        self.ctx_lens = i32(max_requests)
        self.held_blocks = i32(max_requests)
        self.free_blocks = torch.arange(num_blocks, dtype=torch.int32, device=device)
        self.free_head = i32(1)
        self.status = i32(1)
        self._ticket = i32(1)
        self._workspace = attention_workspace(self.device)
        # one for each max_tokens, for as long as the cache lives: captured graphs hold their addresses
        self._plans: Dict[int, PagedStepPlan] = {}
        self._plan: Optional[PagedStepPlan] = None

    def layer(self, index: int):
        """(k_cache, v_cache) of a layer, [num_blocks, block_size, kv_heads, head_dim] views."""
        k, v = self.storage[index]
        return k.transpose(1, 2), v.transpose(1, 2)

    def plan(self, new_lens: torch.Tensor, max_tokens: int) -> PagedStepPlan:
        """Plan a step of ``new_lens`` (int32 [max_requests]) tokens, ``max_tokens`` rows in all; blocks are taken
        for good. Every step of the same ``max_tokens`` writes the same plan, whose tensors live as long as the
        cache does: a CUDA graph that captured them may be replayed between steps of other sizes. A size costs
        8 bytes a token and a request, so a server rounds its sizes up to a few."""
        plan = self._plans.get(max_tokens)
        if plan is None:
            plan = PagedStepPlan.new(self.ctx_lens.numel(), max_tokens, self.device)
            plan.held_blocks, plan.free_head = self.held_blocks, self.free_head
            self._plans[max_tokens] = plan
        self._plan = plan
        return plan_paged_step(self.ctx_lens, new_lens, self.held_blocks, self.free_blocks, self.free_head,
                               self.block_tables, plan, block_size=self.block_size, workspace=self._ticket,
                               status=self.status)

    @property
    def plan_now(self) -> PagedStepPlan:
        """The plan of the step that :meth:`plan` was last called for (a replayed graph has the one it captured)."""
        if self._plan is None:
            raise RuntimeError("PagedKVCache: plan a step first")
        return self._plan

    def write(self, index: int, k: torch.Tensor, v: torch.Tensor) -> None:
        write_paged_kv(k, v, *self.layer(index), self.plan_now.slot_map, status=self.status)

    def attend(self, index: int, q: torch.Tensor, max_q_len: int, *, scale: Optional[float] = None, window: int = 0,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        plan = self.plan_now
        return paged_attention(q, *self.layer(index), self.block_tables, plan.kv_lens, plan.q_indptr,
                               max_q_len=max_q_len, workspace=self._workspace, scale=scale, window=window, out=out,
                               status=self.status)

    def advance(self, num_new: torch.Tensor) -> None:
        """``num_new`` (int32 [max_requests]) of the planned tokens stay in the cache; slots behind them are planned
        again, and their blocks stay with the request."""
        self.ctx_lens.add_(num_new)

    def release(self, requests: Sequence[int]) -> None:
        """Give the blocks of finished requests back and empty their rows (synchronises)."""
        rows: List[int] = sorted(set(int(r) for r in requests))
        if not rows:
            return
        if rows[0] < 0 or rows[-1] >= self.ctx_lens.numel():
            raise IndexError(f"request outside [0, {self.ctx_lens.numel()})")
        held = self.held_blocks[rows].tolist()
        blocks = torch.cat([self.block_tables[r, :n] for r, n in zip(rows, held)])
        head = int(self.free_head.item())
        self.free_blocks[head - blocks.numel():head] = blocks
        self.free_head.sub_(blocks.numel())
        at = torch.tensor(rows, device=self.device)
        self.block_tables[at] = -1
        self.ctx_lens[at] = 0
        self.held_blocks[at] = 0

    def check(self) -> None:
        """Raise if a step so far ran out of blocks or met invalid lengths or tables (synchronises)."""
        check_status(self.status)
