"""Probabilities far below the largest: each is next to nothing in a 16-bit type, together they are not.

P goes in as terms of the cache's type. In f16 what lies below 2^-14 is subnormal; P is scaled so that the largest
lies at 2^11 or above, so terms that are off by half of 2^-24 are off by 2^-36 of the largest each.
"""

from __future__ import annotations

import numpy as np
import pytest

from test_paged_gpu import attend, attention_problem, host, workspace  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu

UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}       # half a unit in the last place, relative
TERMS = {"bf16": 2.0 ** -16, "f16": 2.0 ** -21}     # of P, in two terms


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("requests, q_len, heads, n, power", [
    (1, 1, (1, 1), 60000, 26), (1, 1, (4, 4), 60000, 26), (1, 2, (4, 2), 60000, 26), (1, 40, (1, 1), 60000, 26),
    (1, 300, (1, 1), 60000, 26),
    (10, 1, (32, 32), 2000, 24.5),     # decode kernel, an item in one CTA
    (1, 1, (8, 2), 2000, 24.5),        # a cluster an item
    (40, 20, (32, 8), 2000, 24.5),     # chunk kernel, an item in one CTA
])
def test_one_key_above_tens_of_thousands(cuda_dev, workspace, requests, q_len, heads, n, power, dtype):  # noqa: F811
    """The first key has 2^power times the weight of each other: a small part is theirs, and all of the value."""
    dim, block = 128, 64
    pr = attention_problem(cuda_dev, 72, [q_len] * requests, [n] * requests, *heads, dim, dtype, block)
    scale = dim ** -0.5
    # scores: q = 1 in one column, the first key's there 2^power's logarithm, zeros else (exact in both types but for it)
    pr["q"].zero_()
    pr["q"][..., 0] = 1.0
    pr["k"].zero_()
    pr["v"].copy_(pr["v"].nan_to_num(0.0).abs() + 0.5)
    first = pr["tables"][:, 0].long()
    pr["k"][first, 0, :, 0] = power * np.log(2) / scale
    pr["v"][first, 0] = 0.0
    got = host(attend(pr, workspace)).reshape(requests, q_len, heads[0], dim)
    top = float(pr["k"][first[0], 0, 0, 0]) * scale  # as the type holds it
    seen = np.arange(n - q_len, n)[:, None, None]    # keys besides the first that each row sees
    for i in range(requests):
        v = host(pr["v"][pr["tables"][i, :-(-n // block)].long()]).reshape(-1, heads[1], dim)[:n]
        want = np.repeat(np.cumsum(v, 0)[seen[:, 0, 0]] / (np.exp(top) + seen), heads[0] // heads[1], 1)
        # the result's rounding, P's two terms, the sums' (a sixteenth of n terms after one another), the score's
        bound = (UNIT[dtype] + TERMS[dtype] + 2.0 ** -19 + 2 * top * 2.0 ** -22 + 2 * n * 2.0 ** -24 / 16) * np.abs(want)
        if dtype == "f16":
            bound += n * 2.0 ** -35 * v.max() + 2.0 ** -25
        bad = np.abs(got[i] - want) > bound
        assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4], got[i][bad][:4], want[bad][:4], bound[bad][:4])
