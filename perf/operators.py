"""Timed cases of the paged serving step: block tables and slot maps from request lengths, the cache write,
attention of new tokens over the paged cache, and the verification of drafted tokens.

Every operator is here in two forms. The plain form spells the mathematics out in elementary torch operations,
in 32 bits, rounded once at the end; with ``own`` set, ``run`` calls the library's operators instead. ``exact``
gives the same outputs from the definitions in 64 bits. Request lengths follow from the case alone (a low-discrepancy
spread over its range), so that a case's work does not depend on the seed; contents come from the seed.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
WORKSPACE_BYTES = 64 << 20  # what the library asks of a workspace, whatever the shapes


# --------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # block tables and slots of a decode step: 64 requests with one new token each
        dict(name="plan_decode", op="plan", requests=64, new_lo=1, new_hi=1, ctx_lo=1, ctx_hi=4096, block=16),
        # of a large mixed step: 256 requests with prompts of up to 1024 tokens on contexts of up to 32768
        dict(name="plan_prefill", op="plan", requests=256, new_lo=1, new_hi=1024, ctx_lo=0, ctx_hi=32768, block=16),
        # K and V of one decode step of a model with 32 heads of 128 into the cache
        dict(name="write_decode", op="write", tokens=64, padding=0, q_heads=32, kv_heads=32, dim=128, dtype="bf16",
             block=16, layout="head"),
        # of a prompt batch of 4340 tokens, 8 key heads, read in place from the fused q/k/v projection
        dict(name="write_prefill", op="write", tokens=4340, padding=12, q_heads=32, kv_heads=8, dim=128,
             dtype="bf16", block=16, layout="head"),
        # one request's decode step: latency
        dict(name="attend_one", op="attend", requests=1, q_lo=1, q_hi=1, ctx_lo=776, ctx_hi=776, q_heads=32,
             kv_heads=8, dim=128, dtype="bf16", block=16, window=0, layout="head"),
        # a decode batch of 64 without shared key heads: the cache is the traffic
        dict(name="attend_decode", op="attend", requests=64, q_lo=1, q_hi=1, ctx_lo=33, ctx_hi=2047, q_heads=32,
             kv_heads=32, dim=128, dtype="bf16", block=16, window=0, layout="head"),
        # few requests with long contexts, eight query heads to a key head: the split over the keys
        dict(name="attend_long", op="attend", requests=4, q_lo=1, q_hi=1, ctx_lo=20000, ctx_hi=65535, q_heads=64,
             kv_heads=8, dim=128, dtype="bf16", block=64, window=0, layout="head"),
        # drafts under verification: one to six new tokens for each request
        dict(name="attend_drafts", op="attend", requests=32, q_lo=1, q_hi=6, ctx_lo=1, ctx_hi=8192, q_heads=64,
             kv_heads=8, dim=128, dtype="f16", block=32, window=0, layout="token"),
        # prompts of 128 to 1024 tokens from the start of their cache
        dict(name="attend_prefill", op="attend", requests=8, q_lo=128, q_hi=1024, ctx_lo=0, ctx_hi=0, q_heads=32,
             kv_heads=8, dim=128, dtype="bf16", block=16, window=0, layout="head"),
        # a chunk of a long prompt: 2048 new tokens over 16384 that are in the cache
        dict(name="attend_chunk", op="attend", requests=1, q_lo=2048, q_hi=2048, ctx_lo=16384, ctx_hi=16384,
             q_heads=32, kv_heads=8, dim=128, dtype="bf16", block=16, window=0, layout="head"),
        # three drafted tokens of one request against a small vocabulary: latency
        dict(name="verify_one", op="verify", requests=1, k_lo=3, k_hi=3, vocab=32000, drafter="probs", dtype="f32"),
        # a batch of 256 with up to four drafts each against a large vocabulary
        dict(name="verify_batch", op="verify", requests=256, k_lo=0, k_hi=4, vocab=128256, drafter="probs",
             dtype="f32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "write", "attend", "attend", "attend", "verify"])
    if op == "plan":
        lo, hi = sorted((_log_int(rng, 1, 1024), _log_int(rng, 1, 1024)))
        return dict(op=op, requests=_log_int(rng, 1, 256), new_lo=rng.choice([0, 1, lo]), new_hi=hi,
                    ctx_lo=0, ctx_hi=_log_int(rng, 16, 32768), block=rng.choice([1, 8, 16, 24, 32, 64, 128]))
    if op == "write":
        kv = rng.choice([1, 2, 4, 8, 16, 32])
        return dict(op=op, tokens=_log_int(rng, 1, max(64, 4340 * 8 // kv)), padding=rng.choice([0, 0, 3, 17]),
                    q_heads=kv * rng.choice([1, 4, 8]), kv_heads=kv, dim=rng.choice([64, 128]),
                    dtype=rng.choice(["bf16", "f16", "f32"]), block=rng.choice([8, 16, 24, 32, 64, 128]),
                    layout=rng.choice(["head", "token"]))
    if op == "verify":
        lo, hi = sorted((rng.randint(0, 8), rng.randint(0, 8)))
        return dict(op=op, requests=_log_int(rng, 1, 128), k_lo=lo, k_hi=hi, vocab=_log_int(rng, 1000, 131072),
                    drafter=rng.choice(["probs", "probs", "tokens"]), dtype=rng.choice(["f32", "f32", "bf16", "f16"]))
    most = max(work(c)["bytes"] / 6.5e12 + work(c)["flops"] / 1.6e15 for c in listed() if c["op"] == op)
    while True:
        kv, group = rng.choice([1, 2, 4, 8, 8, 16, 32]), rng.choice([1, 2, 4, 4, 7, 8, 8, 16])
        kind = rng.choice(["decode", "drafts", "prompts", "chunk", "mixed"])
        ctx = sorted((_log_int(rng, 1, 65536), _log_int(rng, 1, 65536)))
        q = {"decode": [1, 1], "drafts": sorted((rng.randint(1, 8), rng.randint(1, 8))),
             "prompts": sorted((_log_int(rng, 9, 2048), _log_int(rng, 9, 2048))),
             "chunk": [_log_int(rng, 65, 4096)] * 2, "mixed": [1, _log_int(rng, 64, 1024)]}[kind]
        requests = 1 if kind == "chunk" else _log_int(rng, 1, 128)
        c = dict(op=op, requests=requests, q_lo=q[0], q_hi=q[1], ctx_lo=0 if kind == "prompts" else ctx[0],
                 ctx_hi=0 if kind == "prompts" else ctx[1], q_heads=kv * group, kv_heads=kv,
                 dim=rng.choice([64, 128, 128]), dtype=rng.choice(["bf16", "f16"]),
                 block=rng.choice([8, 16, 16, 24, 32, 64, 128]), window=rng.choice([0, 0, 0, 4096, 1000]),
                 layout=rng.choice(["head", "token"]))
        w = work(c)
        q_max, kv_max = max(_q_lens(c)), max(_q_lens(c)) + max(_ctx_lens(c))
        padded = requests * kv * group * q_max * kv_max * 4 + requests * kv_max * kv * c["dim"] * 8
        if kv * group <= 128 and w["bytes"] / 6.5e12 + w["flops"] / 1.6e15 < most and padded < 6e9:
            return c


def _spread(lo, hi, n, step):
    """n whole numbers over [lo, hi]: the fractional parts of multiples of an irrational step."""
    return [lo + int((hi - lo + 1) * ((0.5 + i * step) % 1.0)) for i in range(n)]


def _q_lens(c):
    return _spread(c["q_lo"], c["q_hi"], c["requests"], 0.6180339887)


def _ctx_lens(c):
    return _spread(c["ctx_lo"], c["ctx_hi"], c["requests"], 0.7548776662)


def _new_lens(c):
    return _spread(c["new_lo"], c["new_hi"], c["requests"], 0.6180339887)


def _draft_lens(c):
    return _spread(c["k_lo"], c["k_hi"], c["requests"], 0.6180339887)


def _table_width(c):
    return -(-(c["ctx_hi"] + c["new_hi"]) // c["block"]) + 1


def work(case):
    c = case
    if c["op"] == "plan":
        new, ctx, b, r = _new_lens(c), _ctx_lens(c), c["block"], c["requests"]
        fresh = sum(-(-(x + n) // b) - -(-x // b) for x, n in zip(ctx, new))
        touched = sum((x + n - 1) // b - x // b + 1 for x, n in zip(ctx, new) if n)
        # in: three lengths a request, the free blocks taken, the table entries that tokens land in; out: the
        # table entries taken, a slot and a position a token, offsets, lengths and held blocks a request
        return {"bytes": 4 * (3 * r + fresh + (touched - min(touched, fresh)) + fresh + 2 * sum(new) + 3 * r + 4),
                "flops": 0}
    if c["op"] == "write":
        size = torch.empty(0, dtype=DTYPES[c["dtype"]]).element_size()
        return {"bytes": c["tokens"] * (4 * c["kv_heads"] * c["dim"] * size + 4), "flops": 0}
    if c["op"] == "attend":
        seen = keys = 0
        for q, ctx in zip(_q_lens(c), _ctx_lens(c)):
            w = c["window"] or ctx + q
            keys += min(ctx + q, w + q - 1)
            full = max(0, min(q, w - ctx))  # queries that see everything before them
            seen += full * ctx + full * (full + 1) // 2 + (q - full) * w
        rows = 2 * sum(_q_lens(c)) * c["q_heads"] * c["dim"]
        return {"bytes": 2 * (rows + 2 * keys * c["kv_heads"] * c["dim"]) + 4 * keys // c["block"],
                "flops": 4 * seen * c["q_heads"] * c["dim"]}
    size = torch.empty(0, dtype=DTYPES[c["dtype"]]).element_size()
    # the row that the last token is drawn from, and the drafter's beside it where a draft was refused
    # (about two in three drafts pass)
    rows = sum(1 + (c["drafter"] == "probs") * (1 - 0.67 ** k) for k in _draft_lens(c))
    return {"bytes": int(rows * c["vocab"] * size), "flops": int(3 * rows * c["vocab"])}


# -------------------------------------------------------------------------------------------- inputs

def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _indptr(lens):
    return torch.nn.functional.pad(torch.cumsum(_i32(lens), 0), (1, 0)).to(torch.int32)


def _tables(held, width, num_blocks, g):
    """Distinct blocks for every request, in no order: [requests, width] with -1 past a request's own, and the rest."""
    perm = torch.randperm(num_blocks, generator=g, device=DEV, dtype=torch.int32)
    first = torch.cumsum(held, 0) - held
    j = torch.arange(width, device=DEV)
    at = (first[:, None] + j).clamp(max=num_blocks - 1)
    table = torch.where(j < held[:, None], perm[at], torch.full_like(perm[at], -1))
    return table, perm[int(held.sum()):].clone()


def _cache(num_blocks, c, dtype, g):
    """[blocks, block, heads, dim], held token by token or head by head."""
    a, b = (c["block"], c["kv_heads"]) if c["layout"] == "token" else (c["kv_heads"], c["block"])
    t = torch.randn(num_blocks, a, b, c["dim"], generator=g, device=DEV, dtype=dtype)
    return t if c["layout"] == "token" else t.permute(0, 2, 1, 3)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    if c["op"] == "plan":
        new, ctx, b = _i32(_new_lens(c)), _i32(_ctx_lens(c)), c["block"]
        # one request in four holds a block more than its context fills: drafts that were refused
        extra = (torch.rand(c["requests"], generator=g, device=DEV) < 0.25).to(torch.int32)
        held = (ctx + b - 1) // b + extra
        width, tokens = _table_width(c), sum(_new_lens(c))
        num_blocks = sum(-(-(x + n) // b) + 1 for x, n in zip(_ctx_lens(c), _new_lens(c))) + 64
        table, free = _tables(held, width, num_blocks, g)
        r = c["requests"]
        out = dict(q_indptr=torch.empty(r + 1, dtype=torch.int32, device=DEV), kv_lens=torch.empty_like(ctx),
                   held_blocks=torch.empty_like(ctx), free_head=torch.empty(1, dtype=torch.int32, device=DEV),
                   positions=torch.empty(tokens, dtype=torch.int32, device=DEV),
                   slot_map=torch.empty(tokens, dtype=torch.int32, device=DEV))
        return dict(op="plan", ctx_lens=ctx, new_lens=new, held=held, free=free, head=_i32([0]), tables=table,
                    block=b, tokens=tokens, out=out, workspace=torch.zeros(1, dtype=torch.int32, device=DEV))
    if c["op"] == "write":
        dtype, rows = DTYPES[c["dtype"]], c["tokens"] + c["padding"]
        num_blocks = -(-c["tokens"] // c["block"]) * 2 + 1
        slots = torch.randperm(num_blocks * c["block"], generator=g, device=DEV)[:c["tokens"]].to(torch.int32)
        slots = torch.nn.functional.pad(slots, (0, c["padding"]), value=-1)
        heads = c["q_heads"] + 2 * c["kv_heads"]
        qkv = torch.randn(rows, heads, c["dim"], generator=g, device=DEV, dtype=dtype)
        k, v = qkv[:, c["q_heads"]:c["q_heads"] + c["kv_heads"]], qkv[:, c["q_heads"] + c["kv_heads"]:]
        return dict(op="write", k=k, v=v, slots=slots, tokens=c["tokens"], block=c["block"],
                    k_cache=_cache(num_blocks, c, dtype, g), v_cache=_cache(num_blocks, c, dtype, g))
    if c["op"] == "attend":
        dtype, b = DTYPES[c["dtype"]], c["block"]
        q_lens = _q_lens(c)
        kv_lens = [q + x for q, x in zip(q_lens, _ctx_lens(c))]
        held = _i32([-(-n // b) for n in kv_lens])
        num_blocks = sum(-(-n // b) for n in kv_lens) + 8
        table, _ = _tables(held, int(held.max()) + 2, num_blocks, g)
        # scores with a standard deviation of two: attention that is neither flat nor on one key
        q = 2 * torch.randn(sum(q_lens), c["q_heads"], c["dim"], generator=g, device=DEV, dtype=dtype)
        return dict(op="attend", q=q, k_cache=_cache(num_blocks, c, dtype, g), v_cache=_cache(num_blocks, c, dtype, g),
                    tables=table, kv_lens=_i32(kv_lens), q_indptr=_indptr(q_lens), max_q_len=max(q_lens),
                    max_kv_len=max(kv_lens), window=c["window"], scale=c["dim"] ** -0.5,
                    workspace=torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8, device=DEV))
    dtype, lens, v = DTYPES[c["dtype"]], _draft_lens(c), c["vocab"]
    r, k = c["requests"], max(1, c["k_hi"])
    indptr = _indptr([n + 1 for n in lens])
    # logits with heavy tails, and a drafter that is off by some noise
    logits = 2.5 * torch.randn(sum(lens) + r, v, generator=g, device=DEV)
    target = torch.softmax(logits, -1)
    rows = (indptr[:-1, None] + torch.arange(k, device=DEV)).clamp(max=sum(lens) + r - 1).long()
    guess = logits[rows].add_(torch.randn(r, k, v, generator=g, device=DEV), alpha=0.8)
    draft = guess.softmax(-1)
    del logits, guess
    tokens = torch.multinomial(draft.reshape(r * k, v), 1, generator=g).reshape(r, k)
    uniforms = torch.rand(r, k + 1, generator=g, device=DEV)
    return dict(op="verify", target=target.to(dtype), draft=draft.to(dtype) if c["drafter"] == "probs" else None,
                tokens=tokens, indptr=indptr, accept_u=uniforms[:, :k].contiguous(),
                sample_u=uniforms[:, k].contiguous())


# ---------------------------------------------------------------------------------------- plain forms

def _plain_plan(s):
    ctx, new, held, b = s["ctx_lens"], s["new_lens"], s["held"], s["block"]
    width = s["tables"].shape[1]
    end = ctx + new
    wanted = ((end + b - 1) // b).clamp(max=width)
    grant = (wanted - held).clamp(min=0)
    left = s["free"].shape[0] - s["head"]
    upto = torch.cumsum(grant, 0).to(torch.int32)
    first = torch.minimum(upto - grant, left)
    grant = torch.minimum(upto, left) - first
    held_now = held + grant
    j = torch.arange(width, device=DEV, dtype=torch.int32)
    taken = (j >= held[:, None]) & (j < held_now[:, None])
    at = (s["head"] + first[:, None] + j - held[:, None]).clamp(0, s["free"].shape[0] - 1)
    tables = torch.where(taken, s["free"][at.long()], s["tables"])
    q_indptr = torch.cat([torch.zeros_like(s["head"]), torch.cumsum(new, 0).to(torch.int32)])
    t = torch.arange(s["tokens"], device=DEV, dtype=torch.int32)
    req = torch.searchsorted(q_indptr[1:], t, right=True).clamp(max=ctx.shape[0] - 1)
    positions = ctx[req] + t - q_indptr[req]
    page = positions // b
    block = tables[req, page.clamp(max=width - 1)]
    slots = torch.where((page < held_now[req]) & (block >= 0), block * b + positions % b, torch.full_like(t, -1))
    return dict(q_indptr=q_indptr, kv_lens=end, held_blocks=held_now, free_head=s["head"] + grant.sum(0, keepdim=True).to(torch.int32),
                positions=positions, slot_map=slots, block_tables=tables)


def _plain_write(s):
    slots = s["slots"][:s["tokens"]].long()  # the padding at the end has no slot
    s["k_cache"][slots // s["block"], slots % s["block"]] = s["k"][:s["tokens"]]
    s["v_cache"][slots // s["block"], slots % s["block"]] = s["v"][:s["tokens"]]
    return dict(k_cache=s["k_cache"], v_cache=s["v_cache"])


def _plain_attend(s):
    q, kv_lens, indptr = s["q"].float(), s["kv_lens"], s["q_indptr"]
    n, heads, dim = q.shape
    kv_heads, b = s["k_cache"].shape[2], s["k_cache"].shape[1]
    r, q_max, kv_max = kv_lens.shape[0], s["max_q_len"], s["max_kv_len"]
    q_lens = indptr[1:] - indptr[:-1]
    # every request padded to the longest: [requests, heads, queries, keys]
    i, j = torch.arange(q_max, device=DEV), torch.arange(kv_max, device=DEV)
    rows = (indptr[:-1, None] + i).clamp(max=n - 1).long()
    qp = q[rows].reshape(r, q_max, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4)
    qp = qp.reshape(r, kv_heads, (heads // kv_heads) * q_max, dim)
    block = s["tables"][:, j // b].clamp(min=0).long()
    k = s["k_cache"][block, j % b].float().permute(0, 2, 3, 1)
    v = s["v_cache"][block, j % b].float().permute(0, 2, 1, 3)
    scores = torch.matmul(qp * s["scale"], k).reshape(r, heads, q_max, kv_max)
    pos = (kv_lens - q_lens)[:, None] + i
    seen = (j <= pos[..., None]) & (i < q_lens[:, None])[..., None]
    if s["window"]:
        seen &= j > pos[..., None] - s["window"]
    scores = scores.masked_fill_(~seen[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(scores.sub_(top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(r, kv_heads, -1, kv_max), v).reshape(r, heads, q_max, dim)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 2, 1, 3)
    t = torch.arange(n, device=DEV, dtype=torch.int32)
    req = torch.searchsorted(indptr[1:], t, right=True).clamp(max=r - 1)
    return o[req, (t - indptr[req]).long()].to(s["q"].dtype)


def _plain_verify(s):
    target, draft, tokens, indptr = s["target"], s["draft"], s["tokens"], s["indptr"]
    r, k = tokens.shape
    last = target.shape[0] - 1
    each = torch.arange(r, device=DEV)
    count = (indptr[1:] - indptr[:-1] - 1).clamp(max=k)
    i = torch.arange(k, device=DEV)
    rows = (indptr[:-1, None] + i).clamp(max=last).long()
    p = target[rows, tokens].float()
    q = torch.ones_like(p) if draft is None else draft[each[:, None], i, tokens].float()
    passed = (s["accept_u"] * q < p) & (i < count[:, None])
    kept = torch.cumprod(passed.int(), 1).sum(1)
    refused = kept < count
    # the row after the last token kept, less the drafter's where a draft was refused
    w = target[(indptr[:-1] + kept).long()].float()
    at = kept.clamp(max=k - 1)
    if draft is None:
        drop = torch.zeros_like(w).scatter_(1, tokens[each, at][:, None], 1.0) * w
    else:
        drop = draft[each, at].float()
    left = torch.where(refused[:, None], w - drop, w)
    # 40-bit fixed point: sums of whole numbers do not depend on their order
    left = (torch.where(left > 0, left.clamp(max=1.0), 0.0) * 2.0 ** 40).long()
    whole = (torch.where(w > 0, w.clamp(max=1.0), 0.0) * 2.0 ** 40).long()
    left = torch.where(left.sum(1, keepdim=True) > 0, left, whole)
    upto = torch.cumsum(left, 1)
    total = upto[:, -1]
    u = (s["sample_u"] * 2.0 ** 24).long().clamp(0, 2 ** 24 - 1)
    place = (total >> 32) * u * 256 + (((total & 0xFFFFFFFF) * u) >> 24)
    drawn = (upto <= place[:, None]).sum(1)
    drawn = torch.where(total > 0, drawn, torch.full_like(drawn, -1))
    j = torch.arange(k + 1, device=DEV)
    out = torch.where(j < kept[:, None], torch.nn.functional.pad(tokens, (0, 1)), torch.full_like(drawn, -1)[:, None])
    out = torch.where(j == kept[:, None], drawn[:, None], out)
    return dict(tokens=out, num_emitted=(kept + 1).to(torch.int32))


def run(state):
    s = state
    if not own:
        return {"plan": _plain_plan, "write": _plain_write, "attend": _plain_attend, "verify": _plain_verify}[s["op"]](s)
    from multi_lora_b200 import paged_kv, speculative

    if s["op"] == "plan":
        out = paged_kv.PagedStepPlan(**s["out"])
        paged_kv.plan_paged_step(s["ctx_lens"], s["new_lens"], s["held"], s["free"], s["head"], s["tables"], out,
                                 block_size=s["block"], workspace=s["workspace"])
        return dict(s["out"], block_tables=s["tables"])
    if s["op"] == "write":
        paged_kv.write_paged_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
        return dict(k_cache=s["k_cache"], v_cache=s["v_cache"])
    if s["op"] == "attend":
        return paged_kv.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], s["q_indptr"],
                                        max_q_len=s["max_q_len"], scale=s["scale"], window=s["window"],
                                        workspace=s["workspace"])
    tokens, emitted = speculative.verify_draft(s["target"], s["draft"], s["tokens"], s["indptr"], s["accept_u"],
                                               s["sample_u"])
    return dict(tokens=tokens, num_emitted=emitted)


# ------------------------------------------------------------------------------- definitions in 64 bits

def exact(case, seed):
    c = case
    s = prepare(c, seed)
    return {"plan": _exact_plan, "write": _exact_write, "attend": _exact_attend, "verify": _exact_verify}[c["op"]](c, s)


def _exact_plan(c, s):
    b, tables, free = c["block"], s["tables"].cpu().tolist(), s["free"].cpu().tolist()
    held, slots, positions, indptr, kv, head = s["held"].cpu().tolist(), [], [], [0], [], 0
    for i, (x, n) in enumerate(zip(_ctx_lens(c), _new_lens(c))):
        while held[i] * b < x + n:
            tables[i][held[i]] = free[head]
            held[i], head = held[i] + 1, head + 1
        positions += range(x, x + n)
        slots += [tables[i][p // b] * b + p % b for p in range(x, x + n)]
        indptr.append(indptr[-1] + n)
        kv.append(x + n)
    return dict(q_indptr=_i32(indptr), kv_lens=_i32(kv), held_blocks=_i32(held), free_head=_i32([head]),
                positions=_i32(positions), slot_map=_i32(slots), block_tables=_i32(tables))


def _exact_write(c, s):
    k, v = s["k_cache"].double(), s["v_cache"].double()
    for cache, new in ((k, s["k"]), (v, s["v"])):
        at = s["slots"][:c["tokens"]].long()
        cache.index_put_((torch.div(at, c["block"], rounding_mode="floor"), at.remainder(c["block"])),
                         new[:c["tokens"]].double())
    return dict(k_cache=k, v_cache=v)


def _exact_attend(c, s):
    group, b = c["q_heads"] // c["kv_heads"], c["block"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    at = 0
    for i, (n, ctx) in enumerate(zip(_q_lens(c), _ctx_lens(c))):
        key = torch.arange(ctx + n, device=DEV)
        page = s["tables"][i].long()[key // b]
        for h in range(c["kv_heads"]):
            k, v = (t[page, key % b, h].double() for t in (s["k_cache"], s["v_cache"]))
            for e in range(h * group, (h + 1) * group):
                score = s["q"][at:at + n, e].double() @ k.T / math.sqrt(c["dim"])
                behind = torch.arange(ctx, ctx + n, device=DEV)[:, None] - key
                hidden = behind < 0
                if c["window"]:
                    hidden |= behind >= c["window"]
                score[hidden] = -math.inf
                out[at:at + n, e] = torch.softmax(score, 1) @ v
        at += n
    return out


def _exact_verify(c, s):
    """Accept draft x with probability min(1, p(x)/q(x)); after the first refusal one token from the normalised
    positive part of p - q, after none one from p; by inversion, at the given uniforms."""
    tokens, emitted = [], []
    ids, au, su = s["tokens"].cpu().tolist(), s["accept_u"].double().cpu().tolist(), s["sample_u"].double().cpu().tolist()
    k_max, row = s["tokens"].shape[1], 0
    for i, count in enumerate(_draft_lens(c)):
        got = []
        while len(got) < count:
            n, x = len(got), ids[i][len(got)]
            p = float(s["target"][row + n, x])
            q = float(s["draft"][i, n, x]) if s["draft"] is not None else 1.0
            if au[i][n] * q >= p:
                break
            got.append(x)
        w = s["target"][row + len(got)].double()
        if len(got) < count:
            q = s["draft"][i, len(got)].double() if s["draft"] is not None else torch.zeros_like(w)
            if s["draft"] is None:
                q[ids[i][len(got)]] = 1.0
            left = (w - q).clamp(min=0)
            w = left if float(left.sum()) > 0 else w
        upto = torch.cumsum(torch.floor(w * 2.0 ** 40), 0)
        place = torch.floor(upto[-1] * (math.floor(su[i] * 2 ** 24) / 2 ** 24))
        got.append(int(torch.searchsorted(upto, place, right=True)) if float(upto[-1]) > 0 else -1)
        tokens.append(got + [-1] * (k_max + 1 - len(got)))
        emitted.append(len(got))
        row += count + 1
    return dict(tokens=torch.tensor(tokens, device=DEV), num_emitted=_i32(emitted))
