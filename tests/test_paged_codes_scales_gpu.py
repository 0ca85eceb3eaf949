"""Attention over a paged cache of e4m3 codes whose scales of V differ by many powers of two, against 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_paged_codes_gpu import attend, problem, values
from test_paged_gpu import host, status_word, workspace  # noqa: F401  (a fixture)
from test_rotary_gpu import HALF, LEAST

from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu

# Of probabilities times their values' scales, half a step: one f16 term for bf16 results, two for f16's, fp32 for fp32's.
TERMS = {"bf16": 2.0 ** -11, "f16": 2.0 ** -22, "f32": 0.0}


def assert_rows(got, pr, dtype, scale=None, window=0):
    """The result's rounding; scores, scales and sums in fp32 (an error of a score is its probability's); probabilities times
    their values' scales as TERMS has them, and in 16 bits no coarser than 2^-36 of the largest scale (what is
    subnormal in f16 is off by 2^-25, beside a largest one of at least 2^11), times a code of at most 448; and fp32's
    own smallest numbers."""
    dim = pr["q"].shape[2]
    scale = scale or dim ** -0.5
    q, k, v = host(pr["q"]), values(pr["k"], pr["ks"]), values(pr["v"], pr["vs"])
    where = pr["tables"].tolist(), pr["kv_lens"].tolist(), pr["indptr"].tolist()
    want, mean, spread, seen = O.attention(q, k, v, *where, scale, window)
    largest = np.nan_to_num(host(pr["vs"])).max()
    rel_p = dim * 2.0 ** -24 * spread + 2.0 ** -20 + (seen + 64) * 2.0 ** -24
    bound = (HALF[dtype] * np.abs(want) + LEAST[dtype] + (TERMS[dtype] + 2 * rel_p) * mean + seen * 448 * 2.0 ** -149
             + (0 if dtype == "f32" else 1) * seen * 448 * 2.0 ** -36 * largest)
    got = host(got)
    assert np.isfinite(got).all()
    bad = np.abs(got - want) > bound
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], np.broadcast_to(bound, want.shape)[bad][:4])


# requests' new tokens and the heads over two key heads: at most 8 rows an item, 16, one tile of 128, and more
ROWS = [(1, 8), (4, 8), (9, 8), (80, 8)]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("q_len, heads", ROWS)
@pytest.mark.parametrize("small", [2.0 ** -120, 2.0 ** -127, 2.0 ** -130, 1e-40, 2.0 ** -149, 0.0])
def test_scales_of_values_below_fp32_s_smallest_normal(cuda_dev, workspace, small, q_len, heads, dtype):  # noqa: F811
    """In every block, in the first one alone, and in some of a tile beside zeros."""
    pr = problem(cuda_dev, 31, [q_len] * 3, [q_len + 200, q_len + 9, q_len + 300], heads, 2, 128, dtype, 16)
    ordinary = pr["vs"].clone()
    status = status_word(cuda_dev)
    for blocks in ("all", "first", "mixed"):
        pr["vs"] = ordinary.clone() if blocks != "all" else torch.full_like(ordinary, small)
        for row in pr["tables"]:
            if blocks == "first":
                pr["vs"][row[0]] = small
            if blocks == "mixed":
                pr["vs"][row[row >= 0]] = 0
                pr["vs"][row[1]] = small
        assert_rows(attend(pr, workspace, status=status), pr, dtype)
    assert status.item() == 0
