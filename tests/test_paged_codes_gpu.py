"""Attention over a paged cache of e4m3 codes with a scale for each block and head, against oracle/paged_oracle.py.

Codes that no request owns are NaN, and so are the scales of blocks that hold none of its keys: what is let through shows.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from test_paged_decode_gpu import example
from test_paged_gpu import DTYPES, SHAPES, host, i32, status_word, workspace  # noqa: F401  (a fixture)
from test_rotary_gpu import E4M3, HALF

from multi_lora_b200 import paged_kv as P
from multi_lora_b200.rotary import RotaryPositions, rotate
from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu


def problem(dev, seed, q_lens, kv_lens, q_heads, kv_heads, dim, dtype, block, layout="head", spare_rows=0, q_scale=2.0,
            spread=1.0):
    """Requests with exactly these lengths; ``spread``: how much the sizes of blocks differ (a power of e)."""
    g = torch.Generator(device=dev).manual_seed(seed)
    r = len(q_lens)
    held = [-(-n // block) for n in kv_lens]
    blocks = sum(held) + 3
    perm = torch.randperm(blocks, generator=g, device=dev).tolist()
    width, tables, at = max(held + [1]) + 2, [], 0
    shape = (blocks, kv_heads, block, dim + (layout == "odd"))
    caches = [torch.full(shape, 0x7F, dtype=torch.uint8, device=dev).view(E4M3)[..., :dim].transpose(1, 2) for _ in range(2)]
    if layout == "token":
        caches = [c.contiguous() for c in caches]
    scales = [torch.full((kv_heads, blocks), float("nan"), device=dev).T for _ in range(2)]
    for n, h in zip(kv_lens, held):
        own = perm[at:at + h]
        tables.append(own + [-1] * (width - h))
        at += h
        if not n:
            continue
        j = torch.arange(n, device=dev)
        page = torch.tensor(own, device=dev)[j // block]
        for c, f in zip(caches, scales):
            # largest codes between 2 and 448, scales that are no powers of two
            f[own] = torch.exp(spread * torch.randn(h, kv_heads, generator=g, device=dev)) / 32
            c[page, j % block] = (32 * torch.randn(n, kv_heads, dim, generator=g, device=dev)).clamp(-448, 448).to(E4M3)
    indptr = [0]
    for n in q_lens:
        indptr.append(indptr[-1] + n)
    fused = torch.randn(indptr[-1] + spare_rows, q_heads + 2 * kv_heads, dim, generator=g, device=dev)
    q = (q_scale * fused).to(DTYPES[dtype])[:, :q_heads]
    return dict(q=q, k=caches[0], v=caches[1], ks=scales[0], vs=scales[1], tables=i32(tables, dev).reshape(r, width),
                kv_lens=i32(kv_lens, dev), indptr=i32(indptr, dev), max_q_len=max(q_lens + [0]))


def attend(pr, workspace, **kw):  # noqa: F811
    return P.paged_attention(pr["q"], pr["k"], pr["v"], pr["tables"], pr["kv_lens"], pr["indptr"],
                             max_q_len=kw.pop("max_q_len", pr["max_q_len"]), workspace=workspace, k_scales=pr["ks"],
                             v_scales=pr["vs"], **kw)


def values(codes, scales):
    return host(codes.float()) * host(scales)[:, None, :, None]


def assert_attention(got, pr, dtype, window=0, scale=None):
    """The result's rounding; scores in fp32 (their error times p is p's), as their scales'; probabilities times their values'
    scales in 11 bits for bf16 results (16 for others), half a step each, and no coarser than 2^-36 of what the largest
    scale could give (f16 with the largest at 2^11 or more: half a step of its subnormals is 2^-25); sums in fp32."""
    dim = pr["q"].shape[2]
    k, v = values(pr["k"], pr["ks"]), values(pr["v"], pr["vs"])
    out, mean, spread, seen = O.attention(host(pr["q"]), k, v, pr["tables"].tolist(), pr["kv_lens"].tolist(),
                                          pr["indptr"].tolist(), scale or dim ** -0.5, window)
    rel_p = dim * 2.0 ** -24 * spread + 2.0 ** -20 + (seen + 64) * 2.0 ** -24
    most = np.nan_to_num(host(pr["vs"])).max() * 448
    bound = HALF[dtype] * np.abs(out) + ((2.0 ** -12 if dtype == "bf16" else 2.0 ** -17) + 2 * rel_p) * mean + seen * most * 2.0 ** -36
    got = host(got)
    assert np.isfinite(got).all()
    bad = np.abs(got - out) > bound
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], out[bad][:4], np.broadcast_to(bound, out.shape)[bad][:4])


IDS = [f"q{s[0]}-kv{s[1]}-h{s[2]}.{s[3]}-d{s[4]}-b{s[5]}".replace(" ", "") for s in SHAPES]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_attention_matches_the_oracle(cuda_dev, workspace, shape, dtype):  # noqa: F811
    pr = problem(cuda_dev, 1, *shape[:5], dtype, shape[5])
    status = status_word(cuda_dev)
    got = attend(pr, workspace, status=status)
    assert_attention(got, pr, dtype)
    assert torch.equal(attend(pr, workspace, status=status), got)  # the same bits again
    assert status.item() == 0


@pytest.mark.parametrize("q_lens, kv_lens, heads, dim, dtype, block", [
    ([300, 130, 700], [3000, 140, 2500], (16, 16), 64, "bf16", 16),
    ([200, 37, 100], [2600, 1900, 3100], (24, 8), 128, "f16", 8),
    ([3] * 40, [40 * i + 3 for i in range(40)], (16, 8), 128, "bf16", 64),
    ([1] * 90, [31 * i for i in range(90)], (8, 8), 64, "f16", 24),
    ([1] * 300, [7 * (i % 97) for i in range(300)], (32, 32), 128, "bf16", 128),
    ([1, 1], [40000, 100], (8, 1), 128, "bf16", 16),
])
def test_attention_with_many_items_and_tiles_a_cta(cuda_dev, workspace, q_lens, kv_lens, heads, dim, dtype, block):  # noqa: F811
    pr = problem(cuda_dev, 10, q_lens, kv_lens, *heads, dim, dtype, block)
    status = status_word(cuda_dev)
    got = attend(pr, workspace, status=status)
    assert status.item() == 0
    assert_attention(got, pr, dtype)
    assert torch.equal(attend(pr, workspace), got)


@pytest.mark.parametrize("q_lens, kv_lens, dtype", [
    ([900, 130, 257, 700, 64, 1000], [900, 1300, 257, 2700, 3000, 1000], "bf16"),
    ([400] * 6, [5000, 400, 3000, 401, 900, 2000], "f16"),
    ([5, 6, 8, 7] * 40, [85, 120, 100, 700, 90, 128, 129, 300] * 20, "f16"),  # many short items a CTA, of one tile of keys and of two
    ([1, 1, 1, 1] * 12, [3000, 17, 900, 5000] * 12, "bf16"),
])
def test_many_calls_give_the_same_bits(cuda_dev, workspace, q_lens, kv_lens, dtype):  # noqa: F811
    """Every CTA at work over many tiles, again and again: what a stage hands on it has read whole."""
    pr = problem(cuda_dev, 14, q_lens, kv_lens, 32, 8, 128, dtype, 16)
    want = attend(pr, workspace)
    out = torch.empty_like(want)
    wrong = torch.zeros((), dtype=torch.bool, device=cuda_dev)
    for _ in range(60):
        attend(pr, workspace, out=out.fill_(float("nan")))
        wrong |= (out != want).any()
    assert not wrong
    if max(q_lens) < 10:  # the oracle takes its time over the others
        assert_attention(want, pr, dtype)


@pytest.mark.parametrize("dim, block, dtype, layout", [
    (128, 16, "f32", "head"), (64, 5, "f32", "token"), (128, 1, "bf16", "token"), (96, 16, "bf16", "head"),
    (112, 16, "f16", "head"), (40, 24, "bf16", "token"), (256, 12, "f16", "token"), (8, 3, "f16", "head"),
    (128, 16, "bf16", "odd"), (64, 16, "f32", "odd"), (48, 32, "f16", "head"), (72, 16, "bf16", "head"),
])
def test_attention_of_other_shapes(cuda_dev, workspace, dim, block, dtype, layout):  # noqa: F811
    for q_lens, kv_lens in (([1, 9, 40], [50, 9, 301]), ([1, 2, 1], [300, 2, 77])):
        pr = problem(cuda_dev, 2, q_lens, kv_lens, 6, 2, dim, dtype, block, layout)
        assert_attention(attend(pr, workspace), pr, dtype)


@pytest.mark.parametrize("window", [1, 7, 64, 100, 1000])
@pytest.mark.parametrize("q_lens, kv_lens, heads", [([1, 3], [500, 90], (8, 2)), ([150, 20], [600, 21], (4, 1))])
def test_attention_window(cuda_dev, workspace, window, q_lens, kv_lens, heads):  # noqa: F811
    """Blocks that fell out of every query's window may be gone from the table, or hold anything."""
    pr = problem(cuda_dev, 3, q_lens, kv_lens, *heads, 128, "bf16", 16)
    for i, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        gone = max(0, kv - n + 1 - window) // 16
        pr["tables"][i, :gone // 2] = -1
        for name in ("ks", "vs"):
            pr[name][pr["tables"][i, gone // 2:gone].long()] = float("nan")
    status = status_word(cuda_dev)
    assert_attention(attend(pr, workspace, window=window, status=status), pr, "bf16", window)
    assert status.item() == 0


@pytest.mark.parametrize("q_lens, kv_lens", [([1, 2], [9, 40]), ([90, 4], [120, 30])])
def test_attention_rows_behind_the_last_request_are_zero(cuda_dev, workspace, q_lens, kv_lens):  # noqa: F811
    pr = problem(cuda_dev, 4, q_lens, kv_lens, 8, 2, 128, "bf16", 16, spare_rows=21)
    out = torch.full_like(pr["q"], float("nan"))
    got = attend(pr, workspace, out=out, max_q_len=max(q_lens) + 50)
    assert got.data_ptr() == out.data_ptr()
    assert (got[sum(q_lens):] == 0).all()
    assert_attention(got, pr, "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("q_len", [1, 100])
def test_scales_far_apart(cuda_dev, workspace, q_len, dtype):  # noqa: F811
    """Values of sizes from 1e-5 to 1e5 in one request, zero scales among them; large scores, and a scale of its own."""
    pr = problem(cuda_dev, 5, [q_len] * 3, [600, 333, 600], 4, 2, 128, dtype, 16, q_scale=8.0, spread=0.3)
    pr["vs"] *= 10.0 ** torch.randint(-5, 2 if dtype == "f16" else 6, pr["vs"].shape, device=cuda_dev,
                                      generator=torch.Generator(device=cuda_dev).manual_seed(1))
    pr["vs"][pr["tables"][0, 3]] = 0
    pr["ks"][pr["tables"][1, 3]] = 0
    assert_attention(attend(pr, workspace, scale=0.3), pr, dtype, scale=0.3)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("q_len", [1, 80])
def test_queries_of_any_size(cuda_dev, workspace, q_len, dtype):  # noqa: F811
    """Rows of 1e-30 to 1e30, and rows whose elements are; keys so small or large that scores are ordinary."""
    pr = problem(cuda_dev, 6, [q_len] * 3, [200, 150, 90], 4, 2, 64, dtype, 16)
    q = pr["q"].float()
    q[0] *= 1e-30  # scores of nothing
    q[q_len:2 * q_len, 1] *= 1e-4
    q[2 * q_len:, :, ::3] *= 1e-6
    pr["q"] = q.to(pr["q"].dtype)
    assert_attention(attend(pr, workspace), pr, dtype)
    big = dict(pr, q=(q * 1e30).to(pr["q"].dtype), ks=pr["ks"] * 1e-30)
    assert_attention(attend(big, workspace), big, dtype)


@pytest.mark.parametrize("q_len", [1, 80])
def test_attention_reports_blocks_outside_the_cache(cuda_dev, workspace, q_len):  # noqa: F811
    pr = problem(cuda_dev, 6, [q_len, q_len], [200, 150], 4, 2, 64, "f16", 16)
    pr["tables"][0, 3] = -1
    pr["tables"][1, 0] = 10 ** 6
    status = status_word(cuda_dev)
    assert_attention(attend(pr, workspace, status=status), pr, "f16")  # such keys count as zeros
    with pytest.raises(RuntimeError, match="block-table"):
        P.check_status(status)


@pytest.mark.parametrize("q_len", [1, 80])
def test_attention_survives_invalid_lengths(cuda_dev, workspace, q_len):  # noqa: F811
    pr = problem(cuda_dev, 7, [q_len] * 3, [100, 100, 100], 4, 2, 128, "bf16", 16)
    status = status_word(cuda_dev)
    bad = dict(pr, kv_lens=i32([-5, 10 ** 9, 100], cuda_dev))
    got = attend(bad, workspace, status=status)
    assert (got[:q_len] == 0).all()
    ok = attend(pr, workspace)
    assert_attention(ok, pr, "bf16")
    with pytest.raises(RuntimeError, match="length"):
        P.check_status(status)
    bad = dict(pr, indptr=i32([0, q_len, q_len, 10 ** 6], cuda_dev))
    got = attend(bad, workspace, status=status)
    torch.testing.assert_close(got[:q_len], ok[:q_len], rtol=2.0 ** -7, atol=2.0 ** -7)
    with pytest.raises(RuntimeError, match="q_indptr"):
        P.check_status(status)


@pytest.mark.parametrize("q_lens, dtype", [([1, 20, 3, 0, 5] * 12, "bf16"), ([1, 20, 3, 0, 5], "f16"), ([1, 20, 3, 0, 5], "f32")])
def test_requests_longer_than_the_host_said(cuda_dev, workspace, q_lens, dtype):  # noqa: F811
    """Rows that are not computed are reported and zeros; those of the kernel that takes any number are computed."""
    kv_lens = [100, 300, 17, 9, 90] * (len(q_lens) // 5)
    pr = problem(cuda_dev, 61, q_lens, kv_lens, 8, 2, 128, dtype, 16, spare_rows=6)
    want = attend(pr, workspace)
    assert_attention(want, pr, dtype)
    out = torch.full_like(pr["q"], float("nan"))
    status = status_word(cuda_dev)
    attend(pr, workspace, max_q_len=1, out=out, status=status)
    at, gone = 0, 0
    for q in q_lens:
        rows = slice(at, at + q)
        if q > 1 and (out[rows] == 0).all():  # more than the kernel that `max_q_len` = 1 chooses has room for
            gone += 1
        else:
            torch.testing.assert_close(out[rows].float(), want[rows].float(), rtol=2.0 ** -7, atol=2.0 ** -7)
        at += q
    assert (out[at:] == 0).all()
    if gone:
        with pytest.raises(RuntimeError, match="length"):
            P.check_status(status)


MASKED = [
    # q_lens, kv_lens, heads, dim, block, window
    ([5, 8, 1, 2], [200, 8, 300, 65], (4, 2), 128, 16, 0),
    ([3, 1, 8, 2] * 4, [3, 1000, 517, 4000] * 4, (4, 2), 64, 16, 0),
    ([6, 2, 4, 8], [600, 40, 130, 9], (4, 2), 128, 32, 5),
    ([7, 1, 3], [3000, 70, 64], (8, 2), 128, 64, 0),
    ([300, 130, 64, 7], [300, 1400, 64, 2000], (8, 2), 128, 16, 0),
    ([520, 257], [2000, 257], (2, 2), 64, 48, 0),
    ([300, 700, 20], [900, 700, 333], (6, 2), 128, 16, 100),
    ([200, 150], [900, 650], (4, 1), 128, 128, 33),
    ([300, 130, 700], [3000, 140, 2500], (16, 16), 64, 16, 0),
    ([40, 9], [301, 9], (6, 2), 96, 12, 0),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("case", MASKED, ids=[f"q{c[0][:4]}-h{c[2]}-d{c[3]}-w{c[5]}".replace(" ", "") for c in MASKED])
def test_nan_reaches_the_rows_that_see_it_and_no_other(cuda_dev, workspace, case, side, dtype):  # noqa: F811
    q_lens, kv_lens, heads, dim, block, window = case
    pr = problem(cuda_dev, 21, q_lens, kv_lens, *heads, dim, dtype, block)
    clean = attend(pr, workspace, window=window)
    assert clean.isfinite().all()
    touched = torch.zeros_like(clean, dtype=torch.bool)
    at, group = 0, heads[0] // heads[1]
    codes = pr[side].view(torch.uint8)
    for i, (q, kv) in enumerate(zip(q_lens, kv_lens)):
        pos = torch.arange(kv - q, kv, device=cuda_dev)
        some = {kv - q + t for t in (1, q // 3, q // 2, q - 1) if t < q}
        if window:
            some |= {kv - q + 1 - window + t for t in (0, q // 2, min(window, q) - 1)}
        for n, j in enumerate(sorted(j for j in some if 0 <= j < kv)):
            sees = (pos >= j) & ((pos - window < j) if window else True)
            h, c = n % heads[1], (7 * n + 3 * i) % dim
            codes[int(pr["tables"][i, j // block]), j % block, h, c] = (0x7F, 0xFF)[n % 2]
            rows = slice(h * group, (h + 1) * group)
            if side == "v":
                touched[at:at + q, rows, c] |= sees[:, None]
            else:
                touched[at:at + q, rows] |= sees[:, None, None]
        at += q
    got = attend(pr, workspace, window=window)
    assert touched.any() and not touched.all()
    assert torch.equal(got.isnan(), touched)
    assert torch.equal(got[~touched], clean[~touched])  # the same bits


def test_attention_on_another_stream_and_in_a_graph(cuda_dev, workspace):  # noqa: F811
    shapes = [([1] * 20, [30 * i + 1 for i in range(20)]), ([70, 3], [700, 900])]
    problems = [problem(cuda_dev, 8, q, kv, 8, 2, 128, "bf16", 16) for q, kv in shapes]
    want = [attend(pr, workspace) for pr in problems]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [attend(pr, workspace) for pr in problems]
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    outs = [torch.empty(w.shape, dtype=w.dtype, device=cuda_dev) for w in want]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for pr, o in zip(problems, outs):
            attend(pr, workspace, out=o)
    problems[0]["kv_lens"].sub_(1)
    graph.replay()
    assert torch.equal(outs[1], want[1])
    assert_attention(outs[0], problems[0], "bf16")


def test_attention_in_a_large_cache(cuda_dev, workspace):  # noqa: F811
    """Blocks whose offsets pass 2^32 codes (4.8 GB a side), appended to and read."""
    blocks, block, heads, dim = 9250, 64, 64, 128
    kc, vc = (torch.empty(blocks, block, heads, dim, dtype=E4M3, device=cuda_dev) for _ in range(2))
    ks, vs = (torch.ones(blocks, heads, device=cuda_dev) for _ in range(2))
    g = torch.Generator(device=cuda_dev).manual_seed(9)
    own = [blocks - 1, 8800, 3]
    for b in own:
        for c in (kc, vc):
            c[b] = torch.randn(block, heads, dim, generator=g, device=cuda_dev).to(E4M3)
    q = torch.randn(2, heads, dim, generator=g, device=cuda_dev).bfloat16()
    P.append_paged_kv(q, q, kc, vc, i32([(blocks - 1) * block + 5, 8800 * block + 63], cuda_dev), k_scales=ks, v_scales=vs)
    pr = dict(q=q, k=kc, v=vc, ks=ks, vs=vs, tables=i32([own], cuda_dev), kv_lens=i32([190], cuda_dev),
              indptr=i32([0, 2], cuda_dev), max_q_len=2)
    got = attend(pr, workspace)
    at = torch.tensor(own, device=cuda_dev)
    small = dict(pr, k=kc.view(torch.uint8)[at].view(E4M3), v=vc.view(torch.uint8)[at].view(E4M3), ks=ks[at], vs=vs[at],
                 tables=i32([[0, 1, 2]], cuda_dev))
    assert torch.equal(small["v"][1, 63].float(), q[1].to(E4M3).float())
    assert_attention(got, small, "bf16")


def test_refusals(cuda_dev, workspace):  # noqa: F811
    pr = problem(cuda_dev, 1, [1, 1], [20, 30], 4, 2, 64, "bf16", 16)
    ok = dict(q=pr["q"], k_cache=pr["k"], v_cache=pr["v"], block_tables=pr["tables"], kv_lens=pr["kv_lens"],
              q_indptr=pr["indptr"], max_q_len=1, workspace=workspace, k_scales=pr["ks"], v_scales=pr["vs"])
    for change, text in [
        (dict(k_scales=pr["ks"].half()), "scales"), (dict(v_scales=pr["vs"][:, :1]), "scales"), (dict(v_scales=pr["vs"].cpu()), "scales"),
        (dict(k_cache=pr["k"].float(), v_cache=pr["v"].float()), "float8"), (dict(v_cache=pr["v"].float()), "share a dtype"),
        (dict(k_scales=None, v_scales=None), "dtype"), (dict(q=pr["q"][:, :3]), "heads"), (dict(q=pr["q"].double()), "dtype"),
        (dict(q=pr["k"].view(torch.uint8)[0, :2].view(E4M3)), "heads|dtype"), (dict(out=pr["q"].float()), "out"),
        (dict(workspace=workspace[:1000]), "workspace"), (dict(window=-1), "window"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            P.paged_attention(**dict(ok, **change))
    with pytest.raises(ValueError, match="together"):
        P.paged_attention(**dict(ok, v_scales=None))


# --------------------------------------------------------------------------------------- the cache object

@pytest.mark.parametrize("codes", [False, True])
def test_cache_object_over_steps(cuda_dev, codes):
    """Prompts and steps that keep some of their tokens, rotated on the way; blocks of a released request begin again."""
    g = torch.Generator(device=cuda_dev).manual_seed(1)
    r, kv_heads, heads, dim, dtype = 3, 2, 8, 128, torch.bfloat16
    rotary = RotaryPositions.new(dim, cuda_dev)
    radians = [10000.0 ** (-2 * i / dim) for i in range(dim // 2)]
    cache = P.PagedKVCache(layers=2, num_blocks=24, block_size=16, kv_heads=kv_heads, head_dim=dim, max_requests=r,
                           max_blocks=8, dtype=E4M3 if codes else dtype, device=cuda_dev)
    past = [[np.zeros((2, 0, kv_heads, dim)) for _ in range(r)] for _ in range(2)]
    steps = [([70, 3, 0], [70, 3, 0]), ([4, 4, 33], [2, 1, 33]), ([1, 5, 1], [1, 5, 0]), ([1, 1, 1], [1, 1, 1]), None,
             ([90, 1, 60], [90, 1, 60]), ([2, 2, 2], [1, 0, 2])]
    for turn, plan in enumerate(steps):
        if plan is None:
            cache.release([0, 2])
            past = [[p if i == 1 else p[:, :0] for i, p in enumerate(layer)] for layer in past]
            continue
        new, keep = plan
        tokens = sum(new)
        cache.plan(i32(new, cuda_dev), tokens)
        starts = np.cumsum([0] + new)
        for layer in range(2):
            qkv = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=g, device=cuda_dev)
            qkv = (qkv * (0.5 if turn % 2 else 2.0)).to(dtype)
            q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)
            q = cache.append(layer, q, k, v, rotary)
            got = host(cache.attend(layer, q, max(new)))
            positions = host(cache.plan_now.positions)
            rows = np.stack([O.rotate(host(k), positions, radians), host(v)])
            for i in range(r):
                at = slice(starts[i], starts[i + 1])
                kv = np.concatenate([past[layer][i], rows[:, at]], 1)
                if new[i]:
                    n = kv.shape[1]
                    pages = [c.reshape(1, n, kv_heads, dim) for c in kv]
                    want, mean, *_ = O.attention(host(q[at]), *pages, [[0]], [n], [0, new[i]], dim ** -0.5)
                    # the cache's own rounding: of keys (its effect on a score is a sum of 128 of them), and of values
                    step = 2.0 ** -4 if codes else 2.0 ** -8
                    assert np.linalg.norm(got[at] - want) <= 2 * step * np.linalg.norm(mean)
                past[layer][i] = kv[:, :kv.shape[1] - new[i] + keep[i]]
        cache.advance(i32(keep, cuda_dev))
        cache.check()


def test_a_captured_step_is_replayed_between_prompts_of_other_sizes(cuda_dev):
    """A cache of codes: a step that plans, appends and attends, as a graph, next to one that does it call by call."""
    r, heads, kv_heads, dim = 3, 4, 2, 64
    g = torch.Generator(device=cuda_dev).manual_seed(12)
    rotary = RotaryPositions.new(dim, cuda_dev)

    class Side:
        def __init__(self):
            self.cache = P.PagedKVCache(layers=2, num_blocks=60, block_size=16, kv_heads=kv_heads, head_dim=dim, max_requests=r,
                                        max_blocks=30, dtype=E4M3, device=cuda_dev)
            self.new = i32([2] * r, cuda_dev)
            self.qkv = torch.zeros(2 * r, heads + 2 * kv_heads, dim, dtype=torch.bfloat16, device=cuda_dev)
            self.out = [torch.zeros(2 * r, heads, dim, dtype=torch.bfloat16, device=cuda_dev) for _ in range(2)]

        def step(self, new, qkv, most, outs):
            self.cache.plan(new, qkv.shape[0])
            for layer, out in enumerate(outs):
                q = self.cache.append(layer, *qkv.split([heads, kv_heads, kv_heads], 1), rotary)
                self.cache.attend(layer, q, most, out=out)
            self.cache.advance(new)

    eager, captured = Side(), Side()
    for side in (eager, captured):
        side.step(side.new, side.qkv, 2, side.out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step(captured.new, captured.qkv, 2, captured.out)
    for lens in ([40, 0, 3], None, [0, 130, 1], [5, 5, 5], None):
        if lens is not None:
            qkv = torch.randn(sum(lens), heads + 2 * kv_heads, dim, generator=g, device=cuda_dev).bfloat16()
            outs = [[torch.empty_like(qkv[:, :heads]) for _ in range(2)] for _ in range(2)]
            for side, out in zip((eager, captured), outs):
                side.step(i32(lens, cuda_dev), qkv, max(lens), out)
            assert all(torch.equal(a, b) for a, b in zip(*outs))
        qkv = torch.randn(eager.qkv.shape, generator=g, device=cuda_dev)
        for side in (eager, captured):
            side.qkv.copy_(qkv)
        eager.step(eager.new, eager.qkv, 2, eager.out)
        graph.replay()
        for a, b in zip([*eager.out, eager.cache.ctx_lens, eager.cache.storage.view(torch.uint8), eager.cache.scale_storage],
                        [*captured.out, captured.cache.ctx_lens, captured.cache.storage.view(torch.uint8),
                         captured.cache.scale_storage]):
            assert torch.equal(a, b)
    eager.cache.check()
    captured.cache.check()


def test_dispatch_modes_and_profilers_see_the_operators(cuda_dev, workspace):  # noqa: F811
    pr = problem(cuda_dev, 2, [1, 2], [20, 30], 4, 2, 64, "bf16", 16)
    rotary, at = RotaryPositions.new(64, cuda_dev), i32([1, 2, 3], cuda_dev)
    slots = i32([0, 1, 2], cuda_dev)
    calls = {
        "rotate": lambda: rotate(pr["q"], at, rotary),
        "append_paged_kv": lambda: P.append_paged_kv(pr["q"][:, :2], pr["q"][:, 2:], pr["k"], pr["v"], slots, positions=at, rotary=rotary,
                                                     q=pr["q"], k_scales=pr["ks"], v_scales=pr["vs"]),
        "paged_attention_8bit": lambda: attend(pr, workspace),
    }
    seen = []

    class Names(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    for name, call in calls.items():
        plain = call()
        with Names():
            again = call()
        assert any(s.startswith(f"mlora.{name}") for s in seen), (name, seen)
        assert torch.equal(plain, again)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as prof:
        for call in calls.values():
            call()
    assert {f"mlora::{name}" for name in calls} <= {e.name for e in prof.events()}


def test_the_decoder_with_a_cache_of_codes(cuda_dev):
    """The example's decoder: with drafts and a cache of codes it runs, and its first logits, whose attention reads the
    codes of the prompt alone, are near those of its own 16-bit cache (an error of 2^-4 a value, averaged over a sum)."""
    model = example.LoRADecoder()
    slots, lens = i32([0, 3], cuda_dev), [40, 90]
    new = i32(lens, cuda_dev)
    ids = torch.arange(sum(lens), device=cuda_dev)
    with torch.inference_mode():
        values, codes = (model.forward(ids, model.cache(2, 100, dtype=t), new, max(lens), slots).double() for t in (None, E4M3))
    assert 0 < (values - codes).norm() < 2.0 ** -3 * values.norm()
    out, _ = example.generate(model, [[1, 2, 3], [4] * 20], [1, 2], 6, 2, torch.zeros(model.vocab, model.vocab, device=cuda_dev),
                              cache_dtype=E4M3)
    assert all(7 <= len(row) <= 19 for row in out)


def test_two_streams_at_once(cuda_dev, workspace):  # noqa: F811
    """Chunks and decode steps side by side, each stream with its own workspace."""
    other = P.attention_workspace(cuda_dev)
    problems = [problem(cuda_dev, 5, [300, 40, 129], [900, 700, 400], 8, 2, 128, "bf16", 16),
                problem(cuda_dev, 6, [1] * 40, list(range(100, 2100, 50)), 8, 2, 128, "f16", 32),
                problem(cuda_dev, 7, [5] * 9, list(range(300, 1200, 100)), 8, 2, 64, "bf16", 16)]
    want = [attend(pr, workspace).clone() for pr in problems]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(10):
        for s, stream, room in ((0, streams[0], workspace), (1, streams[1], other)):
            with torch.cuda.stream(stream):
                for pr in problems[::1 - 2 * s]:
                    got[s].append(attend(pr, room))
    torch.cuda.synchronize()
    for s in range(2):
        for i, out in enumerate(got[s]):
            assert torch.equal(out, want[::1 - 2 * s][i % 3])


@pytest.mark.parametrize("dim", [64, 80, 96, 112, 128])
@pytest.mark.parametrize("q_len", [1, 3, 20, 70])
def test_heads_that_lie_side_by_side(cuda_dev, workspace, dim, q_len):  # noqa: F811
    """Token by token: behind a head's row lies the next head's, whose codes may be NaN."""
    pr = problem(cuda_dev, dim + q_len, [q_len] * 3, [q_len + 5, 200, 513], 8, 4, dim, "bf16", 16, layout="token")
    want = attend(pr, workspace)
    assert_attention(want, pr, "bf16")
    for cache in (pr["k"], pr["v"]):
        cache.view(torch.uint8)[:, :, 1::2] = 0x7F
    got = attend(pr, workspace)
    assert torch.equal(got.view(3 * q_len, 4, 2, dim)[:, ::2], want.view(3 * q_len, 4, 2, dim)[:, ::2])


@pytest.mark.parametrize("requests, active, heads", [
    (40, {0: 1, 39: 2}, (8, 2)), (1500, {0: 1, 31: 1, 32: 4, 33: 1, 64: 2, 500: 1, 1499: 2}, (8, 2)),  # decode kernels
    (30, {3: 7, 29: 9}, (8, 2)), (40, {0: 7, 39: 30}, (8, 2)), (1200, {i: 1 + i % 30 for i in range(0, 1200, 97)}, (8, 2)),
    (30, {3: 70, 29: 40}, (8, 2)), (300, {0: 30, 150: 200, 299: 5}, (8, 2)),  # chunk kernels
])
def test_few_active_among_many(cuda_dev, workspace, requests, active, heads):  # noqa: F811
    q_lens = [active.get(i, 0) for i in range(requests)]
    kv_lens = [q + 37 * i % 900 if q else 5 * (i % 3) for i, q in enumerate(q_lens)]
    pr = problem(cuda_dev, 91, q_lens, kv_lens, *heads, 64, "bf16", 16, spare_rows=2)
    status = status_word(cuda_dev)
    got = attend(pr, workspace, status=status)
    assert status.item() == 0
    assert (got[sum(q_lens):] == 0).all()
    assert_attention(got, pr, "bf16")


@pytest.mark.parametrize("width", [0, 4, 2000])
@pytest.mark.parametrize("rows, most", [(1, 1), (7, 0), (7, 3), (60, 20), (300, 40)])
def test_no_requests_and_rows(cuda_dev, workspace, rows, most, width):  # noqa: F811
    pr = problem(cuda_dev, 1, [1], [20], 8, 2, 128, "bf16", 16)
    q = torch.randn(rows, 8, 128, device=cuda_dev).bfloat16()
    out, status = torch.full_like(q, float("nan")), status_word(cuda_dev)
    attend(dict(pr, q=q, tables=torch.zeros(0, width, dtype=torch.int32, device=cuda_dev), kv_lens=i32([], cuda_dev),
                indptr=i32([0], cuda_dev), max_q_len=most), workspace, out=out, status=status)
    assert (out == 0).all() and status.item() == 0
