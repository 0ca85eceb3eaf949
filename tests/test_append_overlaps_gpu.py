"""Refusals of tensors whose entries share memory, through torch; and what attention may read of such."""

from __future__ import annotations

import pytest
import torch

from test_paged_codes_gpu import attend, problem
from test_paged_gpu import i32, workspace  # noqa: F401  (a fixture)

from multi_lora_b200 import paged_kv as P

pytestmark = pytest.mark.gpu


def test_expanded_scales_are_read_and_not_written(cuda_dev, workspace):  # noqa: F811
    pr = problem(cuda_dev, 41, [1, 3], [40, 70], 4, 2, 64, "bf16", 16)
    one = {name: pr[name][:, :1].nan_to_num(1.0).contiguous() for name in ("ks", "vs")}
    shared = dict(pr, **{name: t.expand(-1, 2) for name, t in one.items()})
    apart = dict(pr, **{name: t.repeat(1, 2) for name, t in one.items()})
    assert torch.equal(attend(shared, workspace), attend(apart, workspace))
    rows = torch.randn(2, 2, 64, device=cuda_dev).bfloat16()
    slots = i32([0, 1], cuda_dev)
    before = [t.clone() for t in (pr["k"].view(torch.uint8), one["ks"])]
    with pytest.raises(RuntimeError, match="share"):
        P.append_paged_kv(rows, rows, pr["k"], pr["v"], slots, k_scales=shared["ks"], v_scales=apart["vs"])
    with pytest.raises(RuntimeError, match="same"):
        P.append_paged_kv(rows, rows, pr["k"], pr["v"], slots, k_scales=apart["ks"], v_scales=apart["ks"])
    assert torch.equal(before[0], pr["k"].view(torch.uint8)) and torch.equal(before[1], one["ks"])
    P.append_paged_kv(rows, rows, pr["k"], pr["v"], slots, k_scales=apart["ks"], v_scales=apart["vs"])
    both = torch.zeros(pr["k"].shape[0], 2, 2, device=cuda_dev)  # side by side: each entry has its place
    P.append_paged_kv(rows, rows, pr["k"], pr["v"], slots, k_scales=both[..., 0], v_scales=both[..., 1])
    assert torch.equal(both[0], torch.stack([apart["ks"][0], apart["vs"][0]], -1)) and (both[1:] == 0).all()
