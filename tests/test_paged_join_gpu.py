"""Requests whose keys many CTAs share: their pieces are joined in two stages."""

from __future__ import annotations

import pytest
import torch

from test_paged_gpu import assert_attention, attend, attention_problem, status_word, workspace  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("q_lens, kv_lens, heads, dim, block, window", [
    ([1], [30000], (1, 1), 128, 16, 0),                # decode kernel: every CTA has a piece
    ([1, 0, 2], [9000, 3, 20011], (8, 1), 64, 32, 0),  # two turns of rows
    ([1], [30000], (2, 1), 128, 64, 20000),
    ([70, 17], [20070, 9017], (1, 1), 128, 24, 0),     # chunk kernel: two, four threads a row
    ([130], [24130], (1, 1), 64, 64, 0),               # two tiles of rows
    ([5], [26005], (16, 1), 128, 16, 0),
    ([100, 3], [7100, 18003], (6, 2), 96, 16, 5000),
])
def test_attention_with_pieces_on_many_ctas(cuda_dev, workspace, q_lens, kv_lens, heads, dim, block, window, dtype):  # noqa: F811
    pr = attention_problem(cuda_dev, 41, q_lens, kv_lens, *heads, dim, dtype, block)
    status = status_word(cuda_dev)
    got = attend(pr, workspace, window=window, status=status)
    assert status.item() == 0
    assert_attention(got, pr, dtype, window)
    for _ in range(5):
        assert torch.equal(attend(pr, workspace, window=window), got)  # whoever is last
    assert (workspace[:4096] == 0).all()  # the tickets are as they were
