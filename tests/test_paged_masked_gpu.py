"""Keys that only some rows of a request see may hold anything: infinities and NaN there reach the rows that see them, and no other."""

from __future__ import annotations

import pytest
import torch

from test_paged_gpu import attend, attention_problem, i32, status_word, workspace  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

CASES = [
    # q_lens, kv_lens, heads, dim, block, window
    ([5, 8, 1, 2], [200, 8, 300, 65], (4, 2), 128, 16, 0),                     # decode kernel, a cluster an item
    ([3, 1, 8, 2] * 4, [3, 1000, 517, 4000] * 4, (4, 2), 64, 16, 0),           # decode kernel, keys dealt out
    ([6, 2, 4, 8], [600, 40, 130, 9], (4, 2), 128, 32, 5),
    ([7, 1, 3], [3000, 70, 64], (8, 2), 128, 64, 0),                           # chunk kernel, one tile of rows
    ([300, 130, 64, 7], [300, 1400, 64, 2000], (8, 2), 128, 16, 0),
    ([520, 257], [2000, 257], (2, 2), 64, 48, 0),                              # one token a row
    ([300, 700, 20], [900, 700, 333], (6, 2), 128, 16, 100),                   # masked from both sides
    ([200, 150], [900, 650], (4, 1), 128, 128, 33),
    ([300, 130, 700], [3000, 140, 2500], (16, 16), 64, 16, 0),                 # many items a CTA
    ([40, 9], [301, 9], (6, 2), 96, 12, 0),                                    # general kernel
]


def positions(q, kv, window):
    """Some keys that are seen by a part of the request's rows."""
    some = {kv - q + t for t in (1, q // 3, q // 2, q - 1) if t < q}
    if window:
        some |= {kv - q + 1 - window + t for t in (0, q // 2, min(window, q) - 1)}
    return sorted(j for j in some if 0 <= j < kv)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"q{c[0][:4]}-h{c[2]}-d{c[3]}-w{c[5]}".replace(" ", ""))
def test_what_a_row_does_not_see_does_not_reach_it(cuda_dev, workspace, case, side, dtype):  # noqa: F811
    q_lens, kv_lens, heads, dim, block, window = case
    pr = attention_problem(cuda_dev, 21, q_lens, kv_lens, *heads, dim, dtype, block)
    clean = attend(pr, workspace, window=window)
    assert clean.isfinite().all()
    touched = torch.zeros_like(clean, dtype=torch.bool)
    at = 0
    group = heads[0] // heads[1]
    for i, (q, kv) in enumerate(zip(q_lens, kv_lens)):
        pos = torch.arange(kv - q, kv, device=cuda_dev)
        for n, j in enumerate(positions(q, kv, window)):
            sees = (pos >= j) & ((pos - window < j) if window else True)
            h, c = n % heads[1], (7 * n + 3 * i) % dim
            page = int(pr["tables"][i, j // block])
            if side == "v":
                pr["v"][page, j % block, h, c] = (float("nan"), float("inf"), float("-inf"))[n % 3]
                touched[at:at + q, h * group:(h + 1) * group, c] |= sees[:, None]
            else:
                pr["k"][page, j % block, h, c] = float("nan")
                touched[at:at + q, h * group:(h + 1) * group] |= sees[:, None, None]
        at += q
    status = status_word(cuda_dev)
    got = attend(pr, workspace, window=window, status=status)
    assert status.item() == 0
    assert touched.any() and not touched.all()
    assert torch.equal(got.isfinite(), ~touched)
    assert torch.equal(got[~touched], clean[~touched])  # the same bits


@pytest.mark.parametrize("heads, n", [((4, 2), 4), ((8, 2), 200)])
def test_one_infinite_value_is_the_result(cuda_dev, workspace, heads, n):  # noqa: F811
    """The formula's own: p * inf + finite = inf for the rows that see it."""
    pr = attention_problem(cuda_dev, 22, [n], [n], *heads, 64, "bf16", 16, q_scale=0.1)
    j = n - 2
    pr["v"][int(pr["tables"][0, j // 16]), j % 16, :, 5] = float("inf")
    got = attend(pr, workspace)
    assert (got[j:, :, 5] == float("inf")).all()
    assert got[:j].isfinite().all() and got[:, :, :5].isfinite().all() and got[:, :, 6:].isfinite().all()
