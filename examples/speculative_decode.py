"""Speculative decoding of many LoRA requests on a paged cache: one small decoder, end to end.

Every request names an adapter slot. A step feeds each request's last token and
its drafts, packed into one batch:

    plan_paged_step   blocks, slots, positions; its q_indptr routes the LoRA segments too
    apply_lora_group  the adapters' deltas on the fused q/k/v projection (and on o)
    append / attend   queries and keys rotated, new keys and values into the cache, attention over it
    verify_draft      which drafts stay, and the token behind them
    advance           the tokens that stay

The weights are random and the drafter is a table of next-token logits, so the text means
nothing; the emitted tokens are distributed as the decoder's own, drafts or not.

    python examples/speculative_decode.py [--requests 8] [--steps 32] [--drafts 4] [--codes]

With --codes the cache holds keys and values as e4m3 codes, in half the memory.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path
from typing import List, Optional

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from multi_lora_b200 import KernelInputMetaData  # noqa: E402
from multi_lora_b200.backend import get_lora_backend  # noqa: E402
from multi_lora_b200.paged_kv import PagedKVCache  # noqa: E402
from multi_lora_b200.rmsnorm import rmsnorm_fwd  # noqa: E402
from multi_lora_b200.rotary import RotaryPositions  # noqa: E402
from multi_lora_b200.speculative import verify_draft  # noqa: E402


class LoRADecoder:
    """Attention layers with LoRA on q, k, v and o, an embedding and a head; random weights."""

    def __init__(self, *, layers=2, hidden=512, q_heads=8, kv_heads=2, vocab=1000, slots=4, rank=16,
                 dtype=torch.bfloat16, device="cuda", seed=0) -> None:
        g = torch.Generator(device=device).manual_seed(seed)

        def rand(*shape, scale):
            return (scale * torch.randn(*shape, generator=g, device=device)).to(dtype)

        self.q_heads, self.kv_heads, self.dim = q_heads, kv_heads, hidden // q_heads
        self.outs = [hidden, kv_heads * self.dim, kv_heads * self.dim]
        self.embed = rand(vocab, hidden, scale=1.0)
        self.head = rand(vocab, hidden, scale=2 * hidden ** -0.5)
        self.norm = torch.ones(hidden, dtype=dtype, device=device)
        self.layers = []
        for _ in range(layers):
            self.layers.append(dict(
                qkv=rand(sum(self.outs), hidden, scale=hidden ** -0.5), o=rand(hidden, hidden, scale=hidden ** -0.5),
                a=[rand(slots, rank, hidden, scale=hidden ** -0.5) for _ in range(4)],
                b=[rand(slots, n, rank, scale=0.5 * rank ** -0.5) for n in (*self.outs, hidden)]))
        self.ranks = torch.full((slots,), rank, dtype=torch.int32, device=device)
        self.scalings = torch.ones(slots, dtype=dtype, device=device)
        self.freqs = 10000.0 ** (-torch.arange(self.dim // 2, device=device) / (self.dim // 2))
        self.rotary = RotaryPositions.from_frequencies(self.freqs.tolist(), device)
        self.dtype, self.device, self.vocab = dtype, torch.device(device), vocab
        self.backend = get_lora_backend("cuda")

    def cache(self, requests: int, max_tokens: int, block_size: int = 16,
              dtype: Optional[torch.dtype] = None) -> PagedKVCache:
        blocks = -(-max_tokens // block_size)
        return PagedKVCache(layers=len(self.layers), num_blocks=requests * blocks, block_size=block_size,
                            kv_heads=self.kv_heads, head_dim=self.dim, max_requests=requests, max_blocks=blocks,
                            dtype=dtype or self.dtype, device=self.device)

    def forward(self, ids: torch.Tensor, cache: PagedKVCache, new_lens: torch.Tensor, max_q_len: int,
                slots: torch.Tensor) -> torch.Tensor:
        """Logits of the packed tokens ``ids`` (request i's next ``new_lens[i]``, adapter slot ``slots[i]``)."""
        plan = cache.plan(new_lens, ids.numel())
        self.backend.set_kernel_input_metadata(KernelInputMetaData(
            bs=new_lens.numel(), seg_lens=new_lens, seg_indptr=plan.q_indptr, weight_indices=slots,
            lora_ranks=self.ranks, scalings=self.scalings, max_len=max_q_len))
        h = self.embed[ids]
        for i, w in enumerate(self.layers):
            x = rmsnorm_fwd(h, self.norm, 1e-6)
            qkv = F.linear(x, w["qkv"])
            self.backend.apply_lora_group(x, w["a"][:3], w["b"][:3], list(qkv.split(self.outs, -1)))
            q, k, v = (t.unflatten(-1, (-1, self.dim)) for t in qkv.split(self.outs, -1))
            q = cache.append(i, q, k, v, self.rotary)
            o = cache.attend(i, q, max_q_len).flatten(1)
            h = h + self.backend.apply_lora(o, w["a"][3], w["b"][3], F.linear(o, w["o"]))
        return F.linear(rmsnorm_fwd(h, self.norm, 1e-6), self.head)


@torch.inference_mode()
def generate(model: LoRADecoder, prompts: List[List[int]], slots: List[int], steps: int, drafts: int,
             drafter: Optional[torch.Tensor], temperature: float = 1.0, seed: int = 0,
             cache_dtype: Optional[torch.dtype] = None):
    """``steps`` steps behind the prompts. ``drafter`` [vocab, vocab]: next-token logits of the draft model (None with
    ``drafts`` = 0). Returns the emitted tokens per request and the share of drafts that was kept."""
    dev, r = model.device, len(prompts)
    g = torch.Generator(device=dev).manual_seed(seed)
    cache = model.cache(r, max(map(len, prompts)) + steps * (drafts + 1) + 1, dtype=cache_dtype)
    slot_ids = torch.tensor(slots, dtype=torch.int32, device=dev)

    def probs(logits):
        return torch.softmax(logits.float() / temperature, -1)

    # the prompts in one ragged batch; every request's first token comes from its last row
    lens = [len(p) for p in prompts]
    new = torch.tensor(lens, dtype=torch.int32, device=dev)
    logits = model.forward(torch.tensor(sum(prompts, []), device=dev), cache, new, max(lens), slot_ids)
    cache.advance(new)
    ends = torch.cumsum(new, 0).long() - 1
    last = torch.multinomial(probs(logits[ends]), 1, generator=g)
    out, kept = [[t] for t in last[:, 0].tolist()], 0
    new = torch.full((r,), drafts + 1, dtype=torch.int32, device=dev)
    for _ in range(steps):
        tokens, q = [last], []
        for _ in range(drafts):
            q.append(probs(drafter[tokens[-1][:, 0]]))
            tokens.append(torch.multinomial(q[-1], 1, generator=g))
        ids = torch.cat(tokens, 1)  # [requests, drafts + 1]
        logits = model.forward(ids.reshape(-1), cache, new, drafts + 1, slot_ids)
        u = torch.rand(r, drafts + 1, generator=g, device=dev)
        emitted, count = verify_draft(probs(logits), torch.stack(q, 1) if q else None, ids[:, 1:].contiguous(),
                                      cache.plan_now.q_indptr, u[:, :drafts].contiguous(), u[:, drafts].contiguous(),
                                      status=cache.status)
        cache.advance(count)
        last = emitted.gather(1, count[:, None].long() - 1)
        for row, t, n in zip(out, emitted.tolist(), count.tolist()):
            row += t[:n]
            kept += n - 1
    cache.check()
    return out, kept / max(1, r * steps * drafts)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--drafts", type=int, default=4)
    ap.add_argument("--codes", action="store_true", help="a cache of e4m3 codes")
    args = ap.parse_args()
    model = LoRADecoder()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, model.vocab, (int(n),), generator=g).tolist()
               for n in torch.randint(3, 200, (args.requests,), generator=g)]
    drafter = (model.embed @ model.head.T).float()  # what the decoder would say without its layers
    out, share = generate(model, prompts, [i % 4 for i in range(args.requests)], args.steps, args.drafts, drafter,
                          cache_dtype=torch.float8_e4m3fn if args.codes else None)
    total = sum(map(len, out))
    print(f"{total} tokens in {args.steps} steps of {args.requests} requests: "
          f"{total / (args.steps * args.requests):.2f} a step, {100 * share:.0f} % of the drafts kept")


if __name__ == "__main__":
    main()
