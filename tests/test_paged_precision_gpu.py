"""What the 16-bit attention kernels lose besides the result's own rounding, against bounds that would notice
probabilities held in one term of the cache's type.

A probability P of the second product goes in as two terms of the cache's type: 16 bits of it for bf16, 21 for f16.
In f16 what lies far below the largest is subnormal; P is scaled so that the largest lies at 2^11 or above, so two
terms that are off by half of 2^-24 each are off by 2^-35 of the largest. Scores are chosen small, so that their own rounding in
fp32 (dim * 2^-24 of the sum of the products' sizes) stays below that.
"""

from __future__ import annotations

import numpy as np
import pytest

from test_paged_gpu import attend, attention_problem, host, workspace  # noqa: F401  (a fixture)

from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu

UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}       # half a unit in the last place, relative
TERMS = {"bf16": 2.0 ** -16, "f16": 2.0 ** -21}     # of P, in two terms


def bound_of(dtype, out, mean, spread, seen, dim, largest_v):
    rel_p = dim * 2.0 ** -24 * spread + 2.0 ** -20 + (seen + 64) * 2.0 ** -24
    bound = UNIT[dtype] * np.abs(out) + (TERMS[dtype] + 2 * rel_p) * mean + 1e-30
    if dtype == "f16":
        bound = bound + 2.0 ** -25 + seen * 2.0 ** -35 * largest_v  # of the result, and of both terms of each P
    return bound


def one_term(args, dtype):
    """The oracle with every probability (of the largest) rounded to the type's significant bits."""
    bits = {"bf16": 8, "f16": 11}[dtype]
    exp = np.exp

    def rounded(x):
        m, e = np.frexp(exp(x))
        return np.ldexp(np.round(m * 2.0 ** bits) * 2.0 ** -bits, e)

    q, k, v, tables, kv_lens, q_indptr, scale = args
    out = np.zeros(q.shape)
    group = q.shape[1] // k.shape[2]
    for i in range(len(kv_lens)):
        for t in range(q_indptr[i], q_indptr[i + 1]):
            keys = np.arange(kv_lens[i] - (q_indptr[i + 1] - t) + 1)
            at = np.asarray(tables[i])[keys // k.shape[1]]
            for h in range(q.shape[1]):
                s = scale * k[at, keys % k.shape[1], h // group] @ q[t, h]
                p = exp(s - s.max())
                out[t, h] = rounded(s - s.max()) @ v[at, keys % k.shape[1], h // group] / p.sum()
    return out


CASES = [
    # q_lens, kv_lens, heads, dim, block
    ([1], [200], (8, 2), 128, 16),                          # decode kernel, a cluster an item
    ([1, 2] * 10, [40, 90] * 10, (8, 2), 64, 16),           # keys dealt out
    ([1], [9000], (1, 1), 128, 16),                         # pieces on many CTAs
    ([20, 3], [100, 60], (8, 2), 128, 32),                  # chunk kernel, one tile of rows
    ([100, 260], [100, 300], (8, 2), 128, 16),              # two
    ([70], [9000], (1, 1), 64, 16),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"q{c[0][:3]}-kv{c[1][:3]}-h{c[2]}-d{c[3]}".replace(" ", ""))
def test_probabilities_keep_two_terms(cuda_dev, workspace, case, dtype):  # noqa: F811
    q_lens, kv_lens, heads, dim, block = case
    pr = attention_problem(cuda_dev, 71, q_lens, kv_lens, *heads, dim, dtype, block, q_scale=0.1)
    args = (host(pr["q"]), host(pr["k"]), host(pr["v"]), pr["tables"].tolist(), pr["kv_lens"].tolist(),
            pr["indptr"].tolist(), dim ** -0.5)
    out, mean, spread, seen = O.attention(*args)
    largest = float(np.nan_to_num(np.abs(args[2])).max())
    bound = bound_of(dtype, out, mean, spread, seen, dim, largest)
    one = one_term(args, dtype)  # the bound would notice: some outputs of one term are outside of it
    assert seen.max() > 100 or (np.abs(one - out) > bound).any()
    got = host(attend(pr, workspace))
    bad = np.abs(got - out) > bound
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:4], got[bad][:4], out[bad][:4], bound[bad][:4])
