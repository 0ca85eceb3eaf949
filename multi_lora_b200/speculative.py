"""Verification of drafted tokens against the target model's probabilities.

The reference decodes one token a step; a drafter that guesses several needs
its guesses checked so that the emitted tokens are distributed as the target's
own. Draft x with drafter probability q(x) is kept with probability
min(1, p(x) / q(x)); the first refusal draws from the normalised positive part
of p - q instead, and a request whose drafts all pass draws one token more
from the target. All random numbers are arguments.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from multi_lora_b200 import _native


def verify_draft(target_probs: torch.Tensor, draft_probs: Optional[torch.Tensor], draft_tokens: torch.Tensor,
                 row_indptr: torch.Tensor, accept_u: torch.Tensor, sample_u: torch.Tensor, *,
                 status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Tokens that each request emits, int64 [R, K + 1] (-1 behind the last one), and how many, int32 [R].

    target_probs  [rows, V] float32, bfloat16 or float16: request i's rows are
                  row_indptr[i] .. row_indptr[i+1] - 1, one for each draft and one more
    draft_probs   [R, K, V] of the same dtype; None for a drafter without probabilities (every draft certain)
    draft_tokens  int64 [R, K]; request i's first row_indptr[i+1] - row_indptr[i] - 1 count
    accept_u      float32 [R, K], sample_u float32 [R], uniform in [0, 1)

    The draw is by inversion over the vocabulary in 40-bit fixed point: the same
    numbers give the same token whatever the order in which the GPU sums.
    ``status`` (int32 [1], see :func:`multi_lora_b200.paged_kv.check_status`)
    collects rows out of range and drafts outside the vocabulary.
    """
    if not target_probs.is_cuda:
        raise RuntimeError("mlora: verify_draft needs CUDA tensors (no CPU path)")
    return _native.direct("verify_draft")(target_probs, draft_probs, draft_tokens, row_indptr, accept_u, sample_u, status)
