"""Infinities and NaN of values that a row sees: its output is what the formula gives, sum p v with p > 0, so an
infinity is that infinity, two of both signs and any NaN are NaN, and no other column notices."""

from __future__ import annotations

import pytest
import torch

from test_paged_gpu import attend, attention_problem, status_word, workspace  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

CASES = [
    # q_lens, kv_lens, heads, dim, block, window
    ([1], [777], (8, 2), 128, 16, 0),                             # decode kernel, a cluster an item
    ([1, 1], [65, 300], (4, 4), 64, 16, 100),
    ([1] * 20, [33 + 41 * i for i in range(20)], (8, 2), 128, 32, 0),   # keys dealt out
    ([1], [30000], (1, 1), 128, 16, 0),                           # pieces of an item on every CTA
    ([2, 1, 3], [900, 70, 64], (8, 2), 96, 16, 0),
    ([30, 1], [3000, 70], (8, 2), 128, 64, 0),                    # chunk kernel, one tile of rows
    ([300, 64, 7], [300, 900, 2000], (8, 2), 128, 16, 0),         # two
    ([200, 150], [900, 650], (4, 1), 64, 128, 333),
    ([70], [20070], (1, 1), 128, 24, 0),                          # joined from many CTAs
]


def marks(q, kv):
    """Keys of a request, from the first to its last new token's own."""
    return sorted({0, kv // 3, kv // 2, (kv - q) // 2, kv - q, kv - q // 2 - 1, kv - 1})


@pytest.mark.parametrize("q_scale", [0.5, 4.0])  # flat, and so steep that p falls below 16-bit types' range
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"q{c[0][:3]}-kv{c[1][:3]}-h{c[2]}-d{c[3]}-w{c[5]}".replace(" ", ""))
def test_infinities_that_a_row_sees_are_its_result(cuda_dev, workspace, case, dtype, q_scale):  # noqa: F811
    q_lens, kv_lens, heads, dim, block, window = case
    pr = attention_problem(cuda_dev, 51, q_lens, kv_lens, *heads, dim, dtype, block, q_scale=q_scale)
    clean = attend(pr, workspace, window=window)
    assert clean.isfinite().all()
    group = heads[0] // heads[1]
    for i, (q, kv) in enumerate(zip(q_lens, kv_lens)):
        for n, j in enumerate(marks(q, kv)):
            for h in range(heads[1]):
                for c, value in (((5 * n + h) % dim, "inf"), ((5 * n + h + 1) % dim, "-inf"), (3, "inf"), (dim - 1, "nan")):
                    if c == dim - 1 and n != 2 or c == 3 and n not in (1, 3):
                        continue
                    pr["v"][int(pr["tables"][i, j // block]), j % block, h, c] = float(value)
    status = status_word(cuda_dev)
    got = attend(pr, workspace, window=window, status=status).double()
    assert status.item() == 0
    want = torch.zeros_like(got)  # the sum of what is not finite among the values that a row sees
    at = 0
    for i, (q, kv) in enumerate(zip(q_lens, kv_lens)):
        keys = torch.arange(kv, device=cuda_dev)
        v = pr["v"][pr["tables"][i].long()[keys // block], keys % block].double()
        odd = torch.where(v.isfinite(), 0.0, v)
        for j in marks(q, kv):
            pos = torch.arange(kv - q, kv, device=cuda_dev)
            sees = (pos >= j) & ((pos - window < j) if window else True)
            add = odd[j].repeat_interleave(group, 0)
            want[at:at + q] += torch.where(sees[:, None, None], add, 0.0)
        at += q
    touched = want != 0
    assert touched.any() and not touched.all()
    assert torch.equal(got[~touched], clean.double()[~touched])  # the same bits
    assert torch.equal(got[touched].nan_to_num(7.0, 8.0, 9.0), want[touched].nan_to_num(7.0, 8.0, 9.0))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("q_len", [1, 20, 200])
def test_a_score_that_is_nan_wins_over_an_infinity(cuda_dev, workspace, q_len, dtype):  # noqa: F811
    pr = attention_problem(cuda_dev, 52, [q_len, q_len], [600, 600], 4, 2, 128, dtype, 16)
    page = int(pr["tables"][0, 5])
    pr["k"][page, 3, 0, 7] = float("nan")
    pr["v"][page, 9, :, 2] = float("inf")
    got = attend(pr, workspace)
    assert got[:q_len, :2].isnan().all()
    assert (got[:q_len, 2:, 2] == float("inf")).all() and got[:q_len, 2:, 3:].isfinite().all()
    assert got[q_len:].isfinite().all()
