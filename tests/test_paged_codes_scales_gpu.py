"""Attention over a paged cache of e4m3 codes whose scales of V differ by many powers of two, row by row against
64 bits: small values keep their bits, and what a row does not see does not round it."""

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


def peaks(q, keys, v_scales, tables, kv_lens, q_indptr, scale, window=0):
    """Of each row [T, Hq, 1]: the largest probability times its value's scale, what its small values stand beside; and the sum of
    these over keys whose probability is below 2^-112 of the largest one: it may not be fp32's, or 2^128 is below what
    its scale is multiplied by, since the product is below 2^16."""
    tokens, heads, _ = q.shape
    _, block, kv_heads, _ = keys.shape
    out, lost, group = np.zeros((tokens, heads, 1)), np.zeros((tokens, heads, 1)), heads // kv_heads
    for i, kv in enumerate(kv_lens):
        for t in range(q_indptr[i], q_indptr[i + 1]):
            pos = kv - q_indptr[i + 1] + t
            j = np.arange(max(0, pos - window + 1) if window else 0, pos + 1)
            pages = np.asarray(tables[i])[j // block]
            for h in range(heads):
                s = scale * keys[pages, j % block, h // group] @ q[t, h]
                p = np.exp(s - s.max())
                f = p * v_scales[pages, h // group] / p.sum()
                out[t, h], lost[t, h] = f.max(), f[p < 2.0 ** -112].sum()
    return out, lost


def assert_rows(got, pr, dtype, scale=None, window=0):
    """The result's rounding; scores, scales and sums in fp32 (an error of a score is its probability's); probabilities times
    their values' scales as TERMS has them, and in 16 bits no coarser than 2^-33 of the row's largest one (what is
    subnormal in f16 is off by 2^-25, beside a largest one of at least 2^8; where an item has up to 16 rows 2^-36 and
    2^11), times a code of at most 448; and fp32's own smallest numbers."""
    dim = pr["q"].shape[2]
    scale = scale or dim ** -0.5
    q, k, v = host(pr["q"]), values(pr["k"], pr["ks"]), values(pr["v"], pr["vs"])
    where = pr["tables"].tolist(), pr["kv_lens"].tolist(), pr["indptr"].tolist()
    want, mean, spread, seen = O.attention(q, k, v, *where, scale, window)
    largest, lost = peaks(q, k, host(pr["vs"]), *where, scale, window)
    rel_p = dim * 2.0 ** -24 * spread + 2.0 ** -20 + (seen + 64) * 2.0 ** -24
    few = pr["max_q_len"] * (q.shape[1] // k.shape[2]) <= 16
    floor = 0 if dtype == "f32" else 2.0 ** -36 if few else 2.0 ** -33
    bound = (HALF[dtype] * np.abs(want) + LEAST[dtype] + (TERMS[dtype] + 2 * rel_p) * mean + seen * 448 * 2.0 ** -149
             + seen * 448 * floor * largest + 448 * lost)
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


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("q_len, heads", ROWS)
def test_scales_of_blocks_that_a_row_does_not_see(cuda_dev, workspace, q_len, heads, dtype):  # noqa: F811
    """Later tokens in blocks of far larger values, and earlier ones that fell out of a window."""
    kv_lens = [16 * 3 + 1 + q_len // 2, 16 * 20 + 1, q_len + 400]
    kv_lens = [max(n, q_len) for n in kv_lens]
    pr = problem(cuda_dev, 32, [q_len] * 3, kv_lens, heads, 2, 128, dtype, 16)
    up = 2.0 ** (45 if dtype != "f16" else 10)
    if dtype == "f16":
        pr["vs"] *= 2.0 ** -40 if q_len == 1 else 2.0 ** -12
    large = pr["vs"].clone()
    for row, n in zip(pr["tables"], kv_lens):
        large[row[(n - 1) // 16]] *= up
        large[row[(n - q_len // 2 - 1) // 16]] *= up
    assert_rows(attend(dict(pr, vs=large), workspace), dict(pr, vs=large), dtype)
    large = pr["vs"].clone()
    for row, n in zip(pr["tables"], kv_lens):  # the last block that the first of the new tokens sees and others do not
        large[row[max(0, n - q_len - 20) // 16]] *= up
    assert_rows(attend(dict(pr, vs=large), workspace, window=21), dict(pr, vs=large), dtype, window=21)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("q_len, heads", ROWS)
@pytest.mark.parametrize("low", [-10.0, -28.0, -45.0, -200.0])
def test_scales_of_keys_that_a_row_hardly_weighs(cuda_dev, workspace, q_len, heads, dtype, low):  # noqa: F811
    """A block of values 2^45 times the others' size (2^30 of f16's), whose keys score about `low`: its share is from almost
    everything to nothing, and what is left of the others has its bits. At the beginning, in the middle, at the end."""
    kv_lens = [q_len + 150, q_len + 700, q_len + 300]
    pr = problem(cuda_dev, 33, [q_len] * 3, kv_lens, heads, 2, 128, dtype, 16)
    pr["q"] = pr["q"].abs()
    if dtype == "f16":
        pr["vs"] *= 2.0 ** -18
    for row, n, at in zip(pr["tables"], kv_lens, (0, 20, (q_len + 300 - q_len) // 16)):
        block = int(row[at])
        pr["k"].view(torch.uint8)[block] = 0xB8  # minus one
        pr["ks"][block] = -low / (128 ** -0.5 * pr["q"].float().sum(-1).mean())
        pr["vs"][block] *= 2.0 ** (30 if dtype == "f16" else 45)
    pr["ks"] *= 0.25
    for row, at in zip(pr["tables"], (0, 20, 300 // 16)):
        pr["ks"][int(row[at])] *= 4
    assert_rows(attend(pr, workspace), pr, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("q_len, heads", ROWS)
def test_scales_of_any_size_side_by_side(cuda_dev, workspace, q_len, heads, dtype):  # noqa: F811
    """From 2^-100 to 2^90 in one request (what f16 can hold), zeros and minus zeros among them, and of keys too."""
    pr = problem(cuda_dev, 34, [q_len] * 4, [q_len + 500, q_len, q_len + 37, q_len + 2000], heads, 2, 128, dtype, 16)
    g = torch.Generator(device=cuda_dev).manual_seed(2)
    lo, hi = (-100, 5) if dtype == "f16" else (-100, 91)
    power = torch.randint(lo, hi, pr["vs"].shape, device=cuda_dev, generator=g)
    pr["vs"] *= torch.where(torch.rand(pr["vs"].shape, device=cuda_dev, generator=g) < 0.2, 0.0, 1.0) * torch.exp2(power.float())
    for i, row in enumerate(pr["tables"]):
        pr["vs"][row[2]] = -0.0
        pr["ks"][row[1]] = -0.0
    status = status_word(cuda_dev)
    assert_rows(attend(pr, workspace, status=status), pr, dtype)
    assert_rows(attend(pr, workspace, scale=1.5, status=status), pr, dtype, scale=1.5)
    assert status.item() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("q_len, heads", ROWS)
def test_scores_far_above_what_whole_numbers_hold(cuda_dev, workspace, q_len, heads, dtype):  # noqa: F811
    """Scores of up to 1e8: one key has all of a row's weight, and its value comes out as it is."""
    pr = problem(cuda_dev, 35, [q_len] * 2, [q_len + 100, q_len + 500], heads, 2, 128, dtype, 16, spread=0.3)
    for scale in (1e4, 1e6):
        got = host(attend(pr, workspace, scale=scale))
        q, k, v = host(pr["q"]), values(pr["k"], pr["ks"]), values(pr["v"], pr["vs"])
        want, *_ = O.attention(q, k, v, pr["tables"].tolist(), pr["kv_lens"].tolist(), pr["indptr"].tolist(), scale)
        assert np.isfinite(got).all()
        bad = np.abs(got - want) > (HALF[dtype] + TERMS[dtype] + 2.0 ** -20) * np.abs(want)
        # two keys within a rounding of one another may change places: a score's is 2^-23 of it, of which scores are all sizes
        assert bad.any(-1).mean() < 0.01


@pytest.mark.parametrize("q_lens, dtype, rows", [([1, 20, 3, 0, 2, 5] * 12, "bf16", 8), ([1, 20, 3, 0, 2], "f16", 8),
                                                 ([1, 20, 3, 0, 2], "f32", 10 ** 9), ([2, 1, 9, 4, 3] * 9, "bf16", 16)])
def test_exactly_what_does_not_fit_is_not_computed(cuda_dev, workspace, q_lens, dtype, rows):  # noqa: F811
    """Requests longer than the host said: four query heads a key head, so many rows an item; the others' rows are the bits that a
    call without the long ones gives."""
    kv_lens = [100 + 31 * i for i in range(len(q_lens))]
    pr = problem(cuda_dev, 62, q_lens, kv_lens, 8, 2, 128, dtype, 16, spare_rows=6)
    most = 1 if rows != 16 else 3
    fits = [q * 4 <= rows for q in q_lens]
    status = status_word(cuda_dev)
    out = torch.full_like(pr["q"], float("nan"))
    attend(pr, workspace, max_q_len=most, out=out, status=status)
    at, keep = 0, []
    for q, fit in zip(q_lens, fits):
        keep += list(range(at, at + q)) if fit else []
        if not fit:
            assert (out[at:at + q] == 0).all()
        at += q
    assert (out[at:] == 0).all()
    assert (status.item() != 0) >= (not all(fits))
    some = [i for i, fit in enumerate(fits) if fit]
    indptr = np.cumsum([0] + [q_lens[i] for i in some]).tolist()
    short = dict(pr, q=pr["q"][keep], tables=pr["tables"][some], kv_lens=pr["kv_lens"][some],
                 indptr=torch.tensor(indptr, dtype=torch.int32, device=cuda_dev))
    assert_rows(out[keep], short, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("q_len, heads", ROWS)
def test_what_a_row_does_not_see_changes_none_of_its_bits(cuda_dev, workspace, q_len, heads, dtype):  # noqa: F811
    """Keys, values and both scales of the last blocks, larger and smaller ones, under earlier tokens."""
    kv_lens = [16 * n + 1 + q_len // 3 for n in (21, -(-q_len // 16), 8, 60)]
    pr = problem(cuda_dev, 36, [q_len] * 4, kv_lens, heads, 2, 128, dtype, 16, q_scale=6.0)
    want = attend(pr, workspace)
    g = torch.Generator(device=cuda_dev).manual_seed(3)
    for keys, values_ in ((4.0, 2.0 ** 6), (0.0, 2.0 ** -9), (0.5, 0.0)):
        other = {name: pr[name].clone() for name in ("k", "v", "ks", "vs")}
        same, at = torch.ones(4 * q_len, dtype=torch.bool, device=cuda_dev), 0
        for row, n in zip(pr["tables"], kv_lens):
            first = (n - 1 - q_len // 3) // 16 * 16  # the key from which on everything is another
            for page in row[first // 16:-(-n // 16)].long().tolist():
                for name in ("k", "v"):
                    codes = other[name].view(torch.uint8)
                    codes[page] = torch.randint(0, 0x7E, codes[page].shape, generator=g, device=cuda_dev).to(torch.uint8)
                other["ks"][page] *= keys
                other["vs"][page] *= values_
            same[at + max(0, first - (n - q_len)):at + q_len] = False
            at += q_len
        got = attend(dict(pr, **other), workspace)
        assert torch.equal(got[same], want[same]) and not torch.equal(got, want)
        assert same.any() == (q_len > 1)
