"""Head dimensions that no kernel is made for: they run as 64 or 128 columns, the rest of them zeros."""

from __future__ import annotations

import pytest
import torch

from test_paged_gpu import assert_attention, attend, attention_problem, status_word, workspace  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

CASES = [
    # q_lens, kv_lens, heads, block
    ([1, 1], [777, 64], (8, 2), 16),                            # decode kernel, a cluster an item
    ([1, 3, 2] * 8, [1000, 65, 2] * 8, (8, 2), 32),             # decode kernel, keys dealt out
    ([70, 6, 300], [500, 1800, 300], (6, 2), 16),               # chunk kernel; Q row by row
    ([129, 260], [129, 1000], (4, 2), 64),                      # chunk kernel; Q by boxes
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("dim", [8, 40, 72, 80, 96, 120])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"q{c[0][:3]}-h{c[2]}".replace(" ", ""))
def test_attention_of_head_dims_between(cuda_dev, workspace, case, dim, layout, dtype):  # noqa: F811
    q_lens, kv_lens, heads, block = case
    pr = attention_problem(cuda_dev, 31, q_lens, kv_lens, *heads, dim, dtype, block, layout, spare_rows=3)
    status = status_word(cuda_dev)
    out = torch.full((pr["q"].shape[0], heads[0], dim + 8), 7.0, device=cuda_dev, dtype=pr["q"].dtype)
    got = attend(pr, workspace, status=status, out=out[:, :, :dim])  # a slice: nothing behind a row is touched
    assert status.item() == 0
    assert (out[:, :, dim:] == 7).all()
    assert (got[sum(q_lens):] == 0).all()
    assert_attention(got, pr, dtype)


@pytest.mark.parametrize("dim, dtype, block", [(256, "bf16", 16), (136, "f16", 8), (128, "f32", 16), (40, "f32", 5)])
@pytest.mark.parametrize("q_lens, kv_lens, heads, window", [
    ([1], [5000], (8, 8), 0),            # a cluster an item
    ([1, 2], [2100, 700], (14, 2), 0),   # seven heads a key head: four and three
    ([2], [3000], (4, 2), 900),
    ([1, 0, 1], [1, 5, 300], (6, 1), 0),
    ([90, 1] * 3, [90, 1500] * 3, (4, 2), 64),
    ([3], [1], (2, 2), 0),               # rows without a key
])
def test_attention_of_large_heads_and_fp32(cuda_dev, workspace, q_lens, kv_lens, heads, window, dim, dtype, block):  # noqa: F811
    pr = attention_problem(cuda_dev, 32, q_lens, kv_lens, *heads, dim, dtype, block)
    status = status_word(cuda_dev)
    got = attend(pr, workspace, window=window, status=status)
    assert status.item() == 0
    assert_attention(got, pr, dtype, window)
    assert torch.equal(attend(pr, workspace, window=window), got)
