"""A padded step that holds no request: every row gives zeros, whichever kernel takes it."""

from __future__ import annotations

import pytest
import torch

from test_paged_gpu import DTYPES, i32, make_cache, status_word, workspace  # noqa: F401  (a fixture)

from multi_lora_b200 import paged_kv as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, dim, block", [("bf16", 128, 16), ("f16", 64, 16), ("f32", 64, 16), ("bf16", 96, 5)])
@pytest.mark.parametrize("width", [0, 4, 256, 2000])      # tables with room for no, few and many keys
@pytest.mark.parametrize("rows, most", [(1, 1), (7, 1), (7, 0), (300, 40)])
def test_no_requests_and_rows(cuda_dev, workspace, rows, most, width, dtype, dim, block):  # noqa: F811
    kc, vc = (make_cache(cuda_dev, 3, block, 2, dim, DTYPES[dtype], "head") for _ in range(2))
    q = torch.randn(rows, 8, dim, device=cuda_dev).to(DTYPES[dtype])
    out = torch.full_like(q, float("nan"))
    status = status_word(cuda_dev)
    P.paged_attention(q, kc, vc, torch.zeros(0, width, dtype=torch.int32, device=cuda_dev), i32([], cuda_dev),
                      i32([0], cuda_dev), max_q_len=most, workspace=workspace, out=out, status=status)
    assert (out == 0).all()
    assert status.item() == 0
