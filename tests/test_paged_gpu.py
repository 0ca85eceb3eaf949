"""Block tables and slots, the cache write, and attention over the paged cache, against oracle/paged_oracle.py.

Everything that no request owns (slots behind a request's last token, free
blocks, unused table entries) holds NaN or -1 in these tests, so that a kernel that lets
it through shows.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from multi_lora_b200 import paged_kv as P
from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
ROUND = {"bf16": 2.0 ** -9, "f16": 2.0 ** -11, "f32": 2.0 ** -24}  # half a unit in the last place, relative


def i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def status_word(dev):
    return torch.zeros(1, dtype=torch.int32, device=dev)


@pytest.fixture(scope="module")
def workspace(cuda_dev):
    return P.attention_workspace(cuda_dev)


# ------------------------------------------------------------------------------------------------ plan

def run_plan(dev, ctx, new, held, free, head, tables, block, max_tokens, status=None):
    plan = P.PagedStepPlan.new(len(ctx), max_tokens, dev)
    t = i32(tables, dev).reshape(len(ctx), -1)
    P.plan_paged_step(i32(ctx, dev), i32(new, dev), i32(held, dev), i32(free, dev), i32([head], dev), t, plan,
                      block_size=block, workspace=status_word(dev), status=status)
    return dict(q_indptr=plan.q_indptr.tolist(), kv_lens=plan.kv_lens.tolist(), held=plan.held_blocks.tolist(),
                head=plan.free_head.item(), tables=t.tolist(), positions=plan.positions.tolist(),
                slots=plan.slot_map.tolist())


def plan_problem(seed, requests, new_max, ctx_max, block, spare=0, extra=0):
    rng = np.random.default_rng(seed)
    ctx = rng.integers(0, ctx_max + 1, requests).tolist()
    new = (rng.integers(0, new_max + 1, requests) * (rng.random(requests) < 0.8)).tolist()
    held = [-(-c // block) + int(e) for c, e in zip(ctx, rng.integers(0, 2, requests))]
    width = max([-(-(c + n) // block) for c, n in zip(ctx, new)] + held) + extra
    need = sum(max(-(-(c + n) // block) - h, 0) for c, n, h in zip(ctx, new, held))
    blocks = rng.permutation(sum(held) + need + spare + 3).tolist()
    tables, at = [], 0
    for h in held:
        tables.append(blocks[at:at + h] + [-1] * (width - h))
        at += h
    return ctx, new, held, blocks[at:], tables, sum(new)


@pytest.mark.parametrize("requests, new_max, ctx_max, block", [
    (1, 1, 0, 16), (1, 5, 17, 16), (7, 1, 100, 16), (64, 6, 300, 32), (33, 700, 50, 24), (600, 3, 40, 8),
    (513, 40, 9, 1), (5, 9000, 1, 128), (1300, 2, 7, 3),
])
def test_plan_matches_the_oracle(cuda_dev, requests, new_max, ctx_max, block):
    ctx, new, held, free, tables, tokens = plan_problem(requests + new_max, requests, new_max, ctx_max, block)
    status = status_word(cuda_dev)
    for pad in (0, 37):
        got = run_plan(cuda_dev, ctx, new, held, free, 0, tables, block, tokens + pad, status)
        assert got == O.plan(ctx, new, held, free, 0, tables, block, tokens + pad)
    assert status.item() == 0


def test_plan_with_a_used_free_list_and_a_table_view(cuda_dev):
    ctx, new, held, free, tables, tokens = plan_problem(5, 40, 30, 60, 16)
    used = [7] * 11 + free  # 11 entries taken before
    wide = torch.full((40, len(tables[0]) + 9), -5, dtype=torch.int32, device=cuda_dev)
    view = wide[:, 4:4 + len(tables[0])]
    view.copy_(i32(tables, cuda_dev))
    plan = P.PagedStepPlan.new(40, tokens, cuda_dev)
    P.plan_paged_step(i32(ctx, cuda_dev), i32(new, cuda_dev), i32(held, cuda_dev), i32(used, cuda_dev),
                      i32([11], cuda_dev), view, plan, block_size=16, workspace=status_word(cuda_dev))
    want = O.plan(ctx, new, held, used, 11, tables, 16, tokens)
    assert view.tolist() == want["tables"] and plan.slot_map.tolist() == want["slots"]
    assert plan.free_head.item() == want["head"]
    assert (wide[:, :4] == -5).all() and (wide[:, 4 + view.shape[1]:] == -5).all()


def test_plan_in_place_over_steps(cuda_dev):
    """held_blocks and free_head are their own outputs, over many CTAs: the state of one step feeds the next."""
    rng = np.random.default_rng(3)
    r, block, width = 300, 16, 80
    ctx, held, head, free = [0] * r, [0] * r, 0, rng.permutation(r * width).tolist()
    tables = [[-1] * width for _ in range(r)]
    ctx_d, held_d, head_d, free_d = i32(ctx, cuda_dev), i32(held, cuda_dev), i32([0], cuda_dev), i32(free, cuda_dev)
    tables_d, ticket = i32(tables, cuda_dev), status_word(cuda_dev)
    plan = P.PagedStepPlan.new(r, 20000, cuda_dev)
    plan.held_blocks, plan.free_head = held_d, head_d
    for _ in range(6):
        new = rng.integers(0, 60, r).tolist()
        keep = [int(rng.integers(0, n + 1)) for n in new]  # the others are refused: their slots are planned again
        P.plan_paged_step(ctx_d, i32(new, cuda_dev), held_d, free_d, head_d, tables_d, plan, block_size=block,
                          workspace=ticket)
        want = O.plan(ctx, new, held, free, head, tables, block, 20000)
        assert plan.slot_map.tolist() == want["slots"] and plan.q_indptr.tolist() == want["q_indptr"]
        assert held_d.tolist() == want["held"] and head_d.item() == want["head"] and tables_d.tolist() == want["tables"]
        held, head, tables = want["held"], want["head"], want["tables"]
        ctx = [c + k for c, k in zip(ctx, keep)]
        ctx_d.copy_(i32(ctx, cuda_dev))
    assert ticket.item() == 0


def test_plan_when_blocks_or_table_rows_run_out(cuda_dev):
    ctx, new, held, free, tables, tokens = plan_problem(11, 50, 90, 20, 16)
    status = status_word(cuda_dev)
    for left in (0, 1, len(free) // 2):
        got = run_plan(cuda_dev, ctx, new, held, free[:left], 0, tables, 16, tokens, status)
        assert got == O.plan(ctx, new, held, free[:left], 0, tables, 16, tokens)
        with pytest.raises(RuntimeError, match="free list"):
            P.check_status(status)
        assert status.item() == 0
    narrow = [row[:2] for row in tables]  # rows of two blocks: longer requests are cut off
    held2 = [min(h, 2) for h in held]
    got = run_plan(cuda_dev, ctx, new, held2, free, 0, narrow, 16, tokens, status)
    assert got == O.plan(ctx, new, held2, free, 0, narrow, 16, tokens)
    with pytest.raises(RuntimeError, match="length"):
        P.check_status(status)


def test_plan_clamps_invalid_lengths(cuda_dev):
    status = status_word(cuda_dev)
    got = run_plan(cuda_dev, [-3, 5, 0], [2, -1, 4], [0, 1, 0], [4, 5, 6], 0, [[-1] * 4] * 3, 4, 8, status)
    want = O.plan([0, 5, 0], [2, 0, 4], [0, 1, 0], [4, 5, 6], 0, [[-1] * 4] * 3, 4, 8)
    assert {k: got[k] for k in ("slots", "q_indptr", "held", "head", "tables")} == {
        k: want[k] for k in ("slots", "q_indptr", "held", "head", "tables")}
    with pytest.raises(RuntimeError, match="length"):
        P.check_status(status)
    # more tokens than rows: the offsets stay within the rows, and nothing is written past them
    got = run_plan(cuda_dev, [0, 0], [5, 9], [0, 0], [1, 2, 3, 4, 5, 6], 0, [[-1] * 4] * 2, 4, 7, status)
    assert got["q_indptr"] == [0, 5, 7] and got["slots"] == [4, 5, 6, 7, 8, 12, 13]
    with pytest.raises(RuntimeError, match="length"):
        P.check_status(status)


# ----------------------------------------------------------------------------------------------- write

def make_cache(dev, blocks, block, heads, dim, dtype, layout, fill=float("nan")):
    if layout == "head":
        return torch.full((blocks, heads, block, dim), fill, dtype=dtype, device=dev).transpose(1, 2)
    if layout == "odd":  # rows that no 16-byte piece fits: one element off, padded rows
        flat = torch.full((blocks * block * heads * (dim + 1) + 1,), fill, dtype=dtype, device=dev)
        return flat[1:].view(blocks, block, heads, dim + 1)[..., :dim]
    return torch.full((blocks, block, heads, dim), fill, dtype=dtype, device=dev)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tokens, heads, dim, block, layout, fused", [
    (1, 1, 64, 16, "token", False), (64, 32, 128, 16, "head", True), (333, 8, 128, 24, "head", True),
    (50, 3, 72, 7, "token", True), (41, 2, 5, 1, "token", False), (70, 2, 64, 16, "odd", True),
])
def test_write_places_every_row_and_nothing_else(cuda_dev, dtype, tokens, heads, dim, block, layout, fused):
    g = torch.Generator(device=cuda_dev).manual_seed(tokens)
    dt, blocks = DTYPES[dtype], -(-tokens // block) + 3
    if fused:
        qkv = torch.randn(tokens, 4 * heads, dim, generator=g, device=cuda_dev).to(dt)
        k, v = qkv[:, 2 * heads:3 * heads], qkv[:, 3 * heads:]
    else:
        k, v = (torch.randn(tokens, heads, dim, generator=g, device=cuda_dev).to(dt) for _ in range(2))
    slots = torch.randperm(blocks * block, generator=g, device=cuda_dev)[:tokens].to(torch.int32)
    slots[::5] = -1
    kc, vc = (make_cache(cuda_dev, blocks, block, heads, dim, dt, layout, fill=7.0) for _ in range(2))
    status = status_word(cuda_dev)
    P.write_paged_kv(k, v, kc, vc, slots, status=status)
    for cache, new in ((kc, k), (vc, v)):
        want = np.full((blocks * block, heads, dim), 7.0, np.float32)
        for t, s in enumerate(slots.tolist()):
            if s >= 0:
                want[s] = new[t].float().cpu().numpy()
        assert np.array_equal(cache.float().cpu().numpy().reshape(want.shape), want)
    assert status.item() == 0


def test_write_reports_slots_past_the_cache(cuda_dev):
    kc, vc = (make_cache(cuda_dev, 2, 16, 1, 64, torch.bfloat16, "token", fill=1.0) for _ in range(2))
    k = torch.zeros(3, 1, 64, dtype=torch.bfloat16, device=cuda_dev)
    status = status_word(cuda_dev)
    P.write_paged_kv(k, k, kc, vc, i32([32, 31, 2 ** 31 - 1], cuda_dev), status=status)
    assert (kc.reshape(32, 64)[:31] == 1).all() and (kc.reshape(32, 64)[31] == 0).all()
    with pytest.raises(RuntimeError, match="slot"):
        P.check_status(status)


# ------------------------------------------------------------------------------------------- attention

def attention_problem(dev, seed, q_lens, kv_lens, q_heads, kv_heads, dim, dtype, block, layout="head", spare_rows=0,
                      q_scale=2.0):
    """Requests with exactly these lengths; whatever they do not own is NaN or -1."""
    g = torch.Generator(device=dev).manual_seed(seed)
    dt, r = DTYPES[dtype], len(q_lens)
    held = [-(-n // block) for n in kv_lens]
    blocks = sum(held) + 3
    perm = torch.randperm(blocks, generator=g, device=dev).tolist()
    width, tables, at = max(held + [1]) + 2, [], 0
    kc, vc = (make_cache(dev, blocks, block, kv_heads, dim, dt, layout) for _ in range(2))
    for n, h in zip(kv_lens, held):
        own = perm[at:at + h]
        tables.append(own + [-1] * (width - h))
        at += h
        if n:
            j = torch.arange(n, device=dev)
            page = torch.tensor(own, device=dev)[j // block]
            for c in (kc, vc):
                c[page, j % block] = torch.randn(n, kv_heads, dim, generator=g, device=dev).to(dt)
    indptr = [0]
    for n in q_lens:
        indptr.append(indptr[-1] + n)
    fused = torch.randn(indptr[-1] + spare_rows, q_heads + 2 * kv_heads, dim, generator=g, device=dev)
    q = (q_scale * fused).to(dt)[:, :q_heads]  # a slice: rows of the fused projection
    return dict(q=q, k=kc, v=vc, tables=i32(tables, dev).reshape(r, width), kv_lens=i32(kv_lens, dev),
                indptr=i32(indptr, dev), max_q_len=max(q_lens + [0]))


def attend(pr, workspace, **kw):
    return P.paged_attention(pr["q"], pr["k"], pr["v"], pr["tables"], pr["kv_lens"], pr["indptr"],
                             max_q_len=kw.pop("max_q_len", pr["max_q_len"]), workspace=workspace, **kw)


def host(t):
    return t.double().cpu().numpy()


def assert_attention(got, pr, dtype, window=0, scale=None):
    """Within the roundings that the operator has: the result's own, the probabilities' to the cache's type
    before the second product (both relative), scores in fp32 (their error times p is p's), and sums in fp32."""
    dim = pr["q"].shape[2]
    out, mean, spread, seen = O.attention(host(pr["q"]), host(pr["k"]), host(pr["v"]), pr["tables"].tolist(),
                                          pr["kv_lens"].tolist(), pr["indptr"].tolist(),
                                          scale or dim ** -0.5, window)
    eps = ROUND[dtype]
    rel_p = dim * 2.0 ** -24 * spread + 2.0 ** -20 + (seen + 64) * 2.0 ** -24
    bound = eps * np.abs(out) + (eps + 2 * rel_p) * mean + 1e-30
    if dtype == "f16":  # probabilities below 2^-14 of the largest are subnormal
        bound += seen * 2.0 ** -25 * 8
    got = host(got)
    assert np.isfinite(got).all()
    bad = np.abs(got - out) > bound
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], out[bad][:4], np.broadcast_to(bound, out.shape)[bad][:4])


SHAPES = [
    # q_lens, kv_lens, q_heads, kv_heads, dim, block
    ([1], [1], 1, 1, 128, 16),
    ([1], [777], 8, 2, 128, 16),
    ([1, 1, 1], [1, 64, 65], 4, 4, 64, 16),
    ([1] * 9, [5, 0, 16, 17, 300, 128, 129, 63, 1000], 16, 2, 128, 16),
    ([1, 0, 1], [300, 77, 2], 7, 1, 128, 32),
    ([3, 1, 6, 2], [3, 100, 517, 40], 8, 1, 64, 24),
    ([5, 6, 4], [260, 6, 1030], 16, 2, 128, 64),
    ([4] * 5, [4, 130, 33, 500, 64], 32, 2, 128, 128),
    ([70], [70], 4, 1, 128, 16),
    ([129, 1, 64], [400, 513, 64], 8, 2, 128, 16),
    ([300], [333], 2, 2, 64, 8),
    ([33, 257, 1, 0, 5], [33, 800, 900, 12, 700], 6, 2, 128, 48),
    ([2, 9], [1, 9], 4, 2, 128, 16),       # more new tokens than keys: the first rows see nothing
    ([130, 3], [100, 0], 4, 4, 64, 16),
    ([520], [2000], 1, 1, 128, 256),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"q{s[0]}-kv{s[1]}-h{s[2]}.{s[3]}-d{s[4]}-b{s[5]}".replace(" ", ""))
def test_attention_matches_the_oracle(cuda_dev, workspace, shape, dtype):
    pr = attention_problem(cuda_dev, 1, *shape[:5], dtype, shape[5])
    status = status_word(cuda_dev)
    got = attend(pr, workspace, status=status)
    assert_attention(got, pr, dtype)
    assert torch.equal(attend(pr, workspace, status=status), got)  # the same bits again
    assert status.item() == 0


@pytest.mark.parametrize("q_lens, kv_lens, heads, dim, dtype", [
    ([300, 130, 700], [3000, 140, 2500], (16, 16), 64, "bf16"),  # items of two tiles of rows and of one, in turn
    ([200, 37, 100], [2600, 1900, 3100], (24, 8), 128, "f16"),
    ([3] * 40, [40 * i + 3 for i in range(40)], (16, 8), 128, "bf16"),
    ([1] * 90, [31 * i for i in range(90)], (8, 8), 64, "f16"),
])
def test_attention_with_many_items_and_tiles_a_cta(cuda_dev, workspace, q_lens, kv_lens, heads, dim, dtype):
    """Enough work that every CTA runs through its ring of key tiles many times and over item boundaries."""
    pr = attention_problem(cuda_dev, 10, q_lens, kv_lens, *heads, dim, dtype, 16)
    status = status_word(cuda_dev)
    got = attend(pr, workspace, status=status)
    assert status.item() == 0
    assert_attention(got, pr, dtype)
    assert torch.equal(attend(pr, workspace), got)


@pytest.mark.parametrize("dim, block, dtype, layout", [
    (128, 16, "f32", "head"), (64, 5, "f32", "token"), (128, 1, "bf16", "token"), (96, 16, "bf16", "head"),
    (256, 12, "f16", "token"), (8, 3, "f16", "head"), (128, 16, "bf16", "odd"), (64, 16, "f32", "odd"),
])
def test_attention_of_other_shapes(cuda_dev, workspace, dim, block, dtype, layout):
    pr = attention_problem(cuda_dev, 2, [1, 9, 40], [50, 9, 301], 6, 2, dim, dtype, block, layout)
    assert_attention(attend(pr, workspace), pr, dtype)


@pytest.mark.parametrize("window", [1, 7, 64, 100, 1000])
@pytest.mark.parametrize("q_lens, kv_lens, heads", [([1, 3], [500, 90], (8, 2)), ([150, 20], [600, 21], (4, 1))])
def test_attention_window(cuda_dev, workspace, window, q_lens, kv_lens, heads):
    """Blocks that fell out of every query's window may be gone from the table."""
    pr = attention_problem(cuda_dev, 3, q_lens, kv_lens, *heads, 128, "bf16", 16)
    for i, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        gone = max(0, kv - n + 1 - window) // 16
        pr["tables"][i, :gone] = -1
    status = status_word(cuda_dev)
    assert_attention(attend(pr, workspace, window=window, status=status), pr, "bf16", window)
    assert status.item() == 0


@pytest.mark.parametrize("q_lens, kv_lens", [([1, 2], [9, 40]), ([90, 4], [120, 30])])
def test_attention_rows_behind_the_last_request_are_zero(cuda_dev, workspace, q_lens, kv_lens):
    pr = attention_problem(cuda_dev, 4, q_lens, kv_lens, 8, 2, 128, "bf16", 16, spare_rows=21)
    out = torch.full_like(pr["q"], float("nan"))
    got = attend(pr, workspace, out=out, max_q_len=max(q_lens) + 50)
    assert got.data_ptr() == out.data_ptr()
    assert (got[sum(q_lens):] == 0).all()
    assert_attention(got, pr, "bf16")


@pytest.mark.parametrize("q_len", [1, 100])
def test_attention_large_scores_and_scale(cuda_dev, workspace, q_len):
    """One key far above the others, at the start, in the middle and at the end, and a scale of its own."""
    pr = attention_problem(cuda_dev, 5, [q_len] * 3, [600, 600, 600], 4, 2, 128, "bf16", 16, q_scale=8.0)
    for i, j in enumerate((0, 300, 600 - q_len)):
        pr["k"][pr["tables"][i, j // 16], j % 16] = 4 * pr["q"][i * q_len + q_len - 1, :2].sign()
    assert_attention(attend(pr, workspace, scale=0.3), pr, "bf16", scale=0.3)


@pytest.mark.parametrize("q_len", [1, 80])
def test_attention_reports_blocks_outside_the_cache(cuda_dev, workspace, q_len):
    pr = attention_problem(cuda_dev, 6, [q_len, q_len], [200, 150], 4, 2, 64, "f16", 16)
    pr["tables"][0, 3] = -1
    pr["tables"][1, 0] = 10 ** 6
    status = status_word(cuda_dev)
    assert_attention(attend(pr, workspace, status=status), pr, "f16")  # such keys count as zeros
    with pytest.raises(RuntimeError, match="block-table"):
        P.check_status(status)


@pytest.mark.parametrize("q_len", [1, 80])
def test_attention_survives_invalid_lengths(cuda_dev, workspace, q_len):
    """Lengths past the table, negative lengths, offsets past the rows: reported, nothing read or written out of range."""
    pr = attention_problem(cuda_dev, 7, [q_len] * 3, [100, 100, 100], 4, 2, 128, "bf16", 16)
    status = status_word(cuda_dev)
    bad = dict(pr, kv_lens=i32([-5, 10 ** 9, 100], cuda_dev))
    got = attend(bad, workspace, status=status)
    assert (got[:q_len] == 0).all()
    ok = attend(pr, workspace)
    assert torch.equal(got[2 * q_len:], ok[2 * q_len:])
    with pytest.raises(RuntimeError, match="length"):
        P.check_status(status)
    bad = dict(pr, indptr=i32([0, q_len, q_len, 10 ** 6], cuda_dev))
    got = attend(bad, workspace, status=status)
    assert torch.equal(got[:q_len], ok[:q_len])
    with pytest.raises(RuntimeError, match="q_indptr"):
        P.check_status(status)


def test_attention_on_another_stream_and_in_a_graph(cuda_dev, workspace):
    shapes = [([1] * 20, [30 * i + 1 for i in range(20)]), ([70, 3], [700, 900])]
    problems = [attention_problem(cuda_dev, 8, q, kv, 8, 2, 128, "bf16", 16) for q, kv in shapes]
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
    # the lengths are read on the GPU: a replay with others follows them
    problems[0]["kv_lens"].sub_(1)
    graph.replay()
    assert torch.equal(outs[1], want[1])
    assert_attention(outs[0], problems[0], "bf16")


def test_attention_in_a_large_cache(cuda_dev, workspace):
    """Blocks whose offsets pass 2^32 elements (the cache is 9.7 GB a side)."""
    blocks, block, heads, dim = 9250, 64, 64, 128
    kc = torch.empty(blocks, block, heads, dim, dtype=torch.bfloat16, device=cuda_dev)
    vc = torch.empty_like(kc)
    g = torch.Generator(device=cuda_dev).manual_seed(9)
    own = [blocks - 1, 8800, 3]
    for b in own:
        kc[b] = torch.randn(block, heads, dim, generator=g, device=cuda_dev)
        vc[b] = torch.randn(block, heads, dim, generator=g, device=cuda_dev)
    q = torch.randn(2, heads, dim, generator=g, device=cuda_dev).bfloat16()
    slots = i32([(blocks - 1) * block + 5, 8800 * block + 63], cuda_dev)
    P.write_paged_kv(q, q, kc, vc, slots)
    pr = dict(q=q, k=kc, v=vc, tables=i32([own], cuda_dev), kv_lens=i32([190], cuda_dev),
              indptr=i32([0, 2], cuda_dev), max_q_len=2)
    got = attend(pr, workspace)
    small = dict(pr, k=kc[own], v=vc[own], tables=i32([[0, 1, 2]], cuda_dev))
    assert torch.equal(small["k"][0, 5], q[0]) and torch.equal(small["v"][1, 63], q[1])
    assert_attention(got, small, "bf16")


# -------------------------------------------------------------------------------------------- refusals

def test_refusals(cuda_dev, workspace):
    pr = attention_problem(cuda_dev, 1, [1, 1], [20, 30], 4, 2, 64, "bf16", 16)
    ok = dict(q=pr["q"], k_cache=pr["k"], v_cache=pr["v"], block_tables=pr["tables"], kv_lens=pr["kv_lens"],
              q_indptr=pr["indptr"], max_q_len=1, workspace=workspace)
    for change, text in [
        (dict(q=pr["q"].float()), "dtype"), (dict(q=pr["q"][:, :3]), "heads"), (dict(q=pr["q"][..., :32]), "q must be"),
        (dict(k_cache=pr["k"][..., :32]), "k_cache and v_cache"), (dict(v_cache=pr["v"].half()), "dtype"),
        (dict(block_tables=pr["tables"].long()), "block_tables"), (dict(block_tables=pr["tables"][:1]), "block_tables"),
        (dict(block_tables=pr["tables"][:, ::2]), "block_tables"), (dict(kv_lens=pr["kv_lens"].float()), "kv_lens"),
        (dict(q_indptr=pr["indptr"][:2]), "q_indptr"), (dict(workspace=workspace[:1000]), "workspace"),
        (dict(window=-1), "window"), (dict(out=pr["q"][:1]), "out"), (dict(kv_lens=pr["kv_lens"].cpu()), "kv_lens"),
        (dict(q=pr["q"].transpose(0, 2)), "q must be"), (dict(max_q_len=-1), "at most"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            P.paged_attention(**dict(ok, **change))
    with pytest.raises(RuntimeError, match="CUDA"):
        P.paged_attention(**dict(ok, q=pr["q"].cpu()))
    odd = torch.zeros(2, 2, 60, dtype=torch.bfloat16, device=cuda_dev)
    with pytest.raises(RuntimeError, match="head_dim"):
        c = torch.zeros(4, 16, 2, 60, dtype=torch.bfloat16, device=cuda_dev)
        P.paged_attention(**dict(ok, q=odd, k_cache=c, v_cache=c))
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=cuda_dev)
    slots = i32([0, 1], cuda_dev)
    for bad in [dict(k=k.float()), dict(k=k[:, :1]), dict(slot_map=slots[:1]), dict(slot_map=slots.long()),
                dict(v=k[..., :32]), dict(v_cache=pr["v"][:, :8])]:
        with pytest.raises(RuntimeError):
            P.write_paged_kv(**dict(dict(k=k, v=k, k_cache=pr["k"], v_cache=pr["v"], slot_map=slots), **bad))
    plan = P.PagedStepPlan.new(2, 8, cuda_dev)
    two, one = i32([1, 1], cuda_dev), i32([0], cuda_dev)
    good = dict(ctx_lens=two, new_lens=two, held_blocks=two, free_blocks=i32([4, 5], cuda_dev), free_head=one,
                block_tables=pr["tables"], plan=plan, block_size=16, workspace=one.clone())
    for bad in [dict(block_size=0), dict(new_lens=one), dict(held_blocks=two.long()), dict(free_head=two),
                dict(block_tables=pr["tables"][:1]), dict(workspace=one.float()),
                dict(plan=P.PagedStepPlan.new(3, 8, cuda_dev)), dict(new_lens=two.cpu())]:
        with pytest.raises(RuntimeError):
            P.plan_paged_step(**dict(good, **bad))
    many = i32([0] * 8193, cuda_dev)
    with pytest.raises(RuntimeError, match="8192"):
        P.plan_paged_step(many, many, many, many, one, many[:, None], P.PagedStepPlan.new(8193, 8, cuda_dev),
                          block_size=16, workspace=one.clone())


# --------------------------------------------------------------------------------------- the cache object

def test_cache_object_over_steps(cuda_dev):
    """Prompts, then steps that keep only some of their tokens, then a released request's blocks in use again."""
    g = torch.Generator(device=cuda_dev).manual_seed(1)
    r, kv_heads, heads, dim = 3, 2, 8, 128
    cache = P.PagedKVCache(layers=2, num_blocks=30, block_size=16, kv_heads=kv_heads, head_dim=dim, max_requests=r,
                           max_blocks=8, dtype=torch.bfloat16, device=cuda_dev)
    past = [[(torch.zeros(0, kv_heads, dim), torch.zeros(0, kv_heads, dim)) for _ in range(r)] for _ in range(2)]
    free0 = set(range(30))
    for new, keep in [([70, 3, 0], [70, 3, 0]), ([4, 4, 33], [2, 1, 33]), ([1, 5, 1], [1, 5, 0]), ([1, 1, 1], [1, 1, 1])]:
        tokens = sum(new)
        cache.plan(i32(new, cuda_dev), tokens)
        starts = np.cumsum([0] + new)
        for layer in range(2):
            k, v = (torch.randn(tokens, kv_heads, dim, generator=g, device=cuda_dev).bfloat16() for _ in range(2))
            q = torch.randn(tokens, heads, dim, generator=g, device=cuda_dev).bfloat16()
            cache.write(layer, k, v)
            got = cache.attend(layer, q, max(new)).float().cpu()
            for i in range(r):
                rows = slice(starts[i], starts[i + 1])
                kk, vv = (torch.cat([p, t[rows].float().cpu()]) for p, t in zip(past[layer][i], (k, v)))
                if new[i]:
                    n = kk.shape[0]
                    hidden = torch.arange(n) > torch.arange(n - new[i], n)[:, None]
                    s = torch.einsum("thd,jhd->htj", q[rows].float().cpu(), kk.repeat_interleave(heads // kv_heads, 1))
                    p = (s * dim ** -0.5).masked_fill(hidden, -torch.inf).softmax(-1)
                    want = torch.einsum("htj,jhd->thd", p, vv.repeat_interleave(heads // kv_heads, 1))
                    torch.testing.assert_close(got[rows], want, rtol=2 ** -8, atol=2 ** -7)
                past[layer][i] = (kk[:kk.shape[0] - new[i] + keep[i]], vv[:vv.shape[0] - new[i] + keep[i]])
        cache.advance(i32(keep, cuda_dev))
        cache.check()
        own = [b for row, n in zip(cache.block_tables.tolist(), cache.held_blocks.tolist()) for b in row[:n]]
        assert len(own) == len(set(own)) and set(own) | set(cache.free_blocks[cache.free_head.item():].tolist()) == free0
    assert cache.ctx_lens.tolist() == [74, 10, 34]
    cache.release([0, 2])
    assert cache.held_blocks.tolist()[0] == 0 and cache.ctx_lens.tolist() == [0, 10, 0]
    cache.plan(i32([90, 1, 100], cuda_dev), 191)
    cache.check()
    own = [b for row, n in zip(cache.block_tables.tolist(), cache.held_blocks.tolist()) for b in row[:n]]
    assert len(own) == len(set(own))
    with pytest.raises(IndexError):
        cache.release([3])
