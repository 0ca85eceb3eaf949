"""A decode step of a PagedKVCache captured in a CUDA graph, replayed between prompt steps of other sizes."""

from __future__ import annotations

import pytest
import torch

from test_paged_gpu import i32

from multi_lora_b200 import paged_kv as P
from multi_lora_b200.speculative import verify_draft

pytestmark = pytest.mark.gpu

R, HEADS, KV, DIM, VOCAB = 4, 8, 2, 64, 97


class Side:
    """A cache and the buffers of its captured step: plan, write, attention, verification of one draft a request."""

    def __init__(self, dev):
        self.cache = P.PagedKVCache(layers=2, num_blocks=200, block_size=16, kv_heads=KV, head_dim=DIM, max_requests=R,
                                    max_blocks=40, dtype=torch.bfloat16, device=dev)
        self.new = i32([2] * R, dev)
        self.qkv = torch.zeros(2 * R, HEADS + 2 * KV, DIM, dtype=torch.bfloat16, device=dev)
        self.probs = torch.zeros(2 * R, VOCAB, device=dev)
        self.drafts = torch.zeros(R, 1, dtype=torch.long, device=dev)
        self.u = torch.zeros(R, 1, device=dev)
        self.out = [torch.zeros(2 * R, HEADS, DIM, dtype=torch.bfloat16, device=dev) for _ in range(2)]
        self.tokens = torch.zeros(R, 2, dtype=torch.long, device=dev)
        self.emitted = torch.zeros(R, dtype=torch.int32, device=dev)

    def step(self):
        plan = self.cache.plan(self.new, 2 * R)
        for layer, out in enumerate(self.out):
            self.cache.write(layer, self.qkv[:, HEADS:HEADS + KV], self.qkv[:, HEADS + KV:])
            self.cache.attend(layer, self.qkv[:, :HEADS], 2, out=out)
        tokens, emitted = verify_draft(self.probs, None, self.drafts, plan.q_indptr, self.u, self.u[:, 0].contiguous(),
                                       status=self.cache.status)
        self.tokens.copy_(tokens)
        self.emitted.copy_(emitted)
        self.cache.advance(emitted)

    def prompt(self, lens, qkv):
        n = qkv.shape[0]
        new = i32(lens, qkv.device)
        self.cache.plan(new, n)
        outs = []
        for layer in range(2):
            self.cache.write(layer, qkv[:, HEADS:HEADS + KV], qkv[:, HEADS + KV:])
            outs.append(self.cache.attend(layer, qkv[:, :HEADS], max(lens)))
        self.cache.advance(new)
        return outs


def test_replays_between_prompts_of_other_sizes(cuda_dev):
    g = torch.Generator(device=cuda_dev).manual_seed(5)
    eager, captured = Side(cuda_dev), Side(cuda_dev)
    for side in (eager, captured):  # both have taken the step once before
        side.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step()
    held = []
    for turn, lens in enumerate([[40, 0, 3, 0], [0, 200, 0, 1], None, [5, 5, 5, 5], [0, 0, 300, 0], None]):
        if lens is not None:
            n = sum(lens) + turn  # a few padding rows
            qkv = torch.randn(n, HEADS + 2 * KV, DIM, generator=g, device=cuda_dev).bfloat16()
            for a, b in zip(eager.prompt(lens, qkv), captured.prompt(lens, qkv)):
                assert torch.equal(a, b)
        # whatever a replay would still have to be someone's: small tensors of nonsense
        held += [torch.full((size,), 10 ** 9, dtype=torch.int32, device=cuda_dev) for size in (1, R, R + 1, 2 * R) * 8]
        qkv = torch.randn(eager.qkv.shape, generator=g, device=cuda_dev)
        probs = torch.softmax(torch.randn(eager.probs.shape, generator=g, device=cuda_dev), -1)
        drafts = torch.randint(VOCAB, eager.drafts.shape, generator=g, device=cuda_dev)
        u = torch.rand(eager.u.shape, generator=g, device=cuda_dev) * 0.05
        for side in (eager, captured):
            side.qkv.copy_(qkv)
            side.probs.copy_(probs)
            side.drafts.copy_(drafts)
            side.u.copy_(u)
        eager.step()
        graph.replay()
        for a, b in zip([*eager.out, eager.tokens, eager.emitted, eager.cache.ctx_lens, eager.cache.block_tables,
                         eager.cache.held_blocks, eager.cache.free_head, eager.cache.storage],
                        [*captured.out, captured.tokens, captured.emitted, captured.cache.ctx_lens,
                         captured.cache.block_tables, captured.cache.held_blocks, captured.cache.free_head,
                         captured.cache.storage]):
            assert torch.equal(a, b)
    eager.cache.check()
    captured.cache.check()
    assert all((t == 10 ** 9).all() for t in held)
    assert set(eager.emitted.tolist()) <= {1, 2}
