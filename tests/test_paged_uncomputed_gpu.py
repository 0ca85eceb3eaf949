"""Rows that a call does not compute (a request longer than ``max_q_len`` said, offsets that make no sense) are
reported and give zeros: nothing of what the output held before stays."""

from __future__ import annotations

import pytest
import torch

from test_paged_gpu import assert_attention, attend, attention_problem, i32, status_word, workspace  # noqa: F401  (a fixture)

from multi_lora_b200 import paged_kv as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("copies, dim", [(1, 128), (12, 64), (12, 128)])  # a cluster an item; keys dealt out
def test_requests_longer_than_the_host_said(cuda_dev, workspace, copies, dim, dtype):  # noqa: F811
    """Four heads a key head: up to four tokens fit the 16 rows of the kernel that ``max_q_len`` = 1 chooses."""
    q_lens, kv_lens = [1, 20, 3, 0, 5] * copies, [100, 300, 17, 9, 90] * copies
    pr = attention_problem(cuda_dev, 61, q_lens, kv_lens, 8, 2, dim, dtype, 16, spare_rows=6)
    want = attend(pr, workspace)
    out = torch.full_like(pr["q"], float("nan"))
    status = status_word(cuda_dev)
    attend(pr, workspace, max_q_len=1, out=out, status=status)
    with pytest.raises(RuntimeError, match="length"):
        P.check_status(status)
    at = 0
    for q in q_lens:
        rows = slice(at, at + q)
        if q * 4 > 16:
            assert (out[rows] == 0).all()
        else:
            torch.testing.assert_close(out[rows].float(), want[rows].float(), rtol=2.0 ** -7, atol=2.0 ** -7)
        at += q
    assert (out[at:] == 0).all()


BAD = [({2: 10 ** 6}, {1, 2}), ({-1: 10 ** 6}, {-1}), ({2: 0}, {1}), ({0: -3}, {0}), ({-1: 0}, {-1}),
       ({2: -2 ** 31}, {1, 2})]


@pytest.mark.parametrize("dtype, dim", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("copies", [1, 12])
@pytest.mark.parametrize("q", [1, 90])
def test_rows_of_invalid_offsets(cuda_dev, workspace, q, copies, dtype, dim):  # noqa: F811
    """Rows of requests whose offsets are past the rows, negative or decreasing, and the spare ones, are nobody's."""
    n = 4 * copies
    pr = attention_problem(cuda_dev, 62, [q] * n, [200] * n, 4, 2, dim, dtype, 16, spare_rows=5)
    want = attend(pr, workspace)
    for bad, gone in BAD:
        offsets = pr["indptr"].tolist()
        for i, value in bad.items():
            offsets[i] = value
        out = torch.full_like(pr["q"], float("nan"))
        status = status_word(cuda_dev)
        attend(dict(pr, indptr=i32(offsets, cuda_dev)), workspace, out=out, status=status)
        with pytest.raises(RuntimeError, match="q_indptr"):
            P.check_status(status)
        if bad.get(2) == 0:  # request 2 now has rows 0 .. 3 q - 1, as two others do: theirs are anyone's
            assert out.isfinite().all()
            continue
        for i in range(n):
            rows = slice(i * q, (i + 1) * q)
            if i in gone or i - n in gone:
                assert (out[rows] == 0).all()
                out[rows] = want[rows]
        assert (out[n * q:] == 0).all()
        assert_attention(out, pr, dtype)  # the other requests' rows (the keys are dealt out otherwise without these)


@pytest.mark.parametrize("q", [1, 90])
def test_rows_of_invalid_offsets_in_fp32(cuda_dev, workspace, q):  # noqa: F811
    """The kernel for every shape looks a row's request up in the offsets: where they decrease, any row may give zeros."""
    pr = attention_problem(cuda_dev, 63, [q] * 4, [200] * 4, 4, 2, 64, "f32", 16, spare_rows=5)
    want = attend(pr, workspace)
    for bad, _ in BAD:
        offsets = pr["indptr"].tolist()
        for i, value in bad.items():
            offsets[i] = value
        out = torch.full_like(pr["q"], float("nan"))
        status = status_word(cuda_dev)
        attend(dict(pr, indptr=i32(offsets, cuda_dev)), workspace, out=out, status=status)
        assert out.isfinite().all()
        if bad.get(2) != 0:
            assert ((out == want) | (out == 0)).all()
            with pytest.raises(RuntimeError, match="q_indptr"):
                P.check_status(status)


@pytest.mark.parametrize("requests, tokens, heads, width, block, most", [
    (10, 600, (4, 2), 20, 16, 1),
    (1025, 300, (4, 2), 20, 16, 1),
    (8192, 4096, (64, 8), 1024, 128, 0),  # the key tiles of all requests pass 32 bits: nothing is computed
])
def test_offsets_that_go_back_and_forth(cuda_dev, workspace, requests, tokens, heads, width, block, most):  # noqa: F811
    """Every other request claims all rows: reported, and the rows are anyone's (all values are one) or zeros."""
    k = torch.ones(4, block, heads[1], 64, dtype=torch.bfloat16, device=cuda_dev)
    q = torch.ones(tokens, heads[0], 64, dtype=torch.bfloat16, device=cuda_dev)
    offsets = torch.arange(requests + 1, device=cuda_dev, dtype=torch.int32) % 2 * tokens
    out = torch.full_like(q, float("nan"))
    status = status_word(cuda_dev)
    P.paged_attention(q, k, k, torch.zeros(requests, width, dtype=torch.int32, device=cuda_dev),
                      torch.full((requests,), width * block, dtype=torch.int32, device=cuda_dev), offsets,
                      max_q_len=tokens, workspace=workspace, out=out, status=status)
    assert ((out >= 0) & (out <= most)).all()
    with pytest.raises(RuntimeError, match="q_indptr"):
        P.check_status(status)
