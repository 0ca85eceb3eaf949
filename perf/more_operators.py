"""Timed cases of rotary positions and of a paged cache held in 8 bits: the rotation of queries and keys, the append of
rotated keys and of values to a paged cache in 16 or 32 bits, the same to a cache of e4m3 codes with a scale for each
block and head, and attention of new tokens over such a cache.

Every operator is here in two forms. The plain form spells the mathematics out in elementary torch operations,
in 32 bits (angles in 64), rounded once at the end; with ``own`` set, ``run`` calls the library's operators instead.
``exact`` gives the same outputs from the definitions in 64 bits, codes before they are rounded. Request lengths follow
from the case alone (a low-discrepancy spread over its range), so that a case's work does not depend on the seed;
contents come from the seed.

What the codes stand for: slot s of block b, head h holds codes c with a scale f[b, h], the values c * f. A call that
appends to a block takes f = 2^k with the smallest k for which the largest finite magnitude of its new rows there is at most
448 * 2^k (k >= -100); where the block holds rows before them, not less than the scale that it has, and those rows' codes
follow a scale that grows, rounded to nearest even. Infinities are held as +-448 f.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E4M3 = torch.float8_e4m3fn
MOST = 448.0  # the largest e4m3 value
LEAST = 2.0 ** -100  # the smallest scale
WORKSPACE_BYTES = 64 << 20  # what the library asks of a workspace, whatever the shapes


# --------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # queries of one decode step of 64 requests, 32 heads: latency
        dict(name="rotate_decode", op="rotate", tokens=64, heads=32, dim=128, rotary_dim=128, dtype="bf16",
             interleaved=False, scaling="none", pos_hi=4095),
        # queries of a prompt batch of 4340 tokens on far positions of a model with scaled frequencies, neighbours as pairs
        dict(name="rotate_prefill", op="rotate", tokens=4340, heads=32, dim=128, rotary_dim=128, dtype="bf16",
             interleaved=True, scaling="bands", pos_hi=131071),
        # one decode step of 64 requests: queries rotated, keys rotated into a 16-bit cache, values beside them
        dict(name="append_decode", op="append", requests=64, new_lo=1, new_hi=1, ctx_lo=1, ctx_hi=4095, padding=0, q_heads=32,
             kv_heads=8, dim=128, rotary_dim=128, dtype="bf16", interleaved=False, scaling="none", block=16, layout="head", bits=16),
        # the same of a prompt batch of 4340 tokens
        dict(name="append_prefill", op="append", requests=8, new_lo=61, new_hi=1023, ctx_lo=0, ctx_hi=0, padding=12,
             q_heads=32, kv_heads=8, dim=128, rotary_dim=128, dtype="bf16", interleaved=False, scaling="bands", block=16,
             layout="head", bits=16),
        # a large decode step of 512 requests into an 8-bit cache: one row in each block, most of them begun earlier
        dict(name="append8_decode", op="append", requests=512, new_lo=1, new_hi=1, ctx_lo=1, ctx_hi=4095, padding=0, q_heads=64,
             kv_heads=8, dim=128, rotary_dim=128, dtype="bf16", interleaved=False, scaling="bands", block=16, layout="head", bits=8),
        # a prompt batch into an 8-bit cache
        dict(name="append8_prefill", op="append", requests=8, new_lo=61, new_hi=1023, ctx_lo=0, ctx_hi=0, padding=12,
             q_heads=32, kv_heads=8, dim=128, rotary_dim=128, dtype="bf16", interleaved=False, scaling="none", block=32,
             layout="head", bits=8),
        # one request's decode step over an 8-bit cache: latency
        dict(name="attend8_one", op="attend", requests=1, q_lo=1, q_hi=1, ctx_lo=900, ctx_hi=900, q_heads=32,
             kv_heads=8, dim=128, dtype="bf16", block=16, window=0, layout="head"),
        # a decode batch of 96 without shared key heads: the cache is the traffic
        dict(name="attend8_decode", op="attend", requests=96, q_lo=1, q_hi=1, ctx_lo=33, ctx_hi=4095, q_heads=32,
             kv_heads=32, dim=128, dtype="bf16", block=16, window=0, layout="head"),
        # few requests with long contexts, eight query heads to a key head: the split over the keys
        dict(name="attend8_long", op="attend", requests=4, q_lo=1, q_hi=1, ctx_lo=40000, ctx_hi=131071, q_heads=64,
             kv_heads=8, dim=128, dtype="bf16", block=64, window=0, layout="head"),
        # drafts under verification: one to six new tokens for each request
        dict(name="attend8_drafts", op="attend", requests=32, q_lo=1, q_hi=6, ctx_lo=1, ctx_hi=8192, q_heads=64,
             kv_heads=8, dim=128, dtype="f16", block=32, window=0, layout="token"),
        # prompts of 128 to 1024 tokens from the start of their cache
        dict(name="attend8_prefill", op="attend", requests=8, q_lo=128, q_hi=1024, ctx_lo=0, ctx_hi=0, q_heads=32,
             kv_heads=8, dim=128, dtype="bf16", block=16, window=0, layout="head"),
        # a chunk of a long prompt: 2048 new tokens over 16384 that are in the cache
        dict(name="attend8_chunk", op="attend", requests=1, q_lo=2048, q_hi=2048, ctx_lo=16384, ctx_hi=16384,
             q_heads=32, kv_heads=8, dim=128, dtype="bf16", block=16, window=0, layout="head"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15


def _rotary_draw(rng):
    dim = rng.choice([64, 72, 96, 128, 128, 128, 256])
    return dict(dim=dim, rotary_dim=rng.choice([dim, dim, dim, dim // 2 // 2 * 2, 32]), interleaved=rng.choice([False, False, True]),
                scaling=rng.choice(["none", "bands", "linear"]))


def draw(rng):
    op = rng.choice(["rotate", "append", "append", "attend", "attend", "attend"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        if op == "rotate":
            c = dict(op=op, tokens=_log_int(rng, 1, 8192), heads=rng.choice([1, 2, 8, 20, 32, 64]),
                     dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), pos_hi=_log_int(rng, 100, 1000000), **_rotary_draw(rng))
        elif op == "append":
            kv, bits = rng.choice([1, 2, 3, 4, 8, 8, 16, 32]), rng.choice([8, 8, 16])
            prompts = rng.choice([False, True])
            new = sorted((_log_int(rng, 1, 1024), _log_int(rng, 1, 1024))) if prompts else sorted((rng.randint(0, 8), rng.randint(1, 8)))
            ctx = sorted((_log_int(rng, 1, 16384), _log_int(rng, 1, 16384)))
            c = dict(op=op, requests=_log_int(rng, 1, 16 if prompts else 512), new_lo=new[0], new_hi=new[1], ctx_lo=rng.choice([0, ctx[0]]),
                     ctx_hi=ctx[1], padding=rng.choice([0, 0, 3, 17]), q_heads=kv * rng.choice([1, 4, 8]), kv_heads=kv,
                     dtype=rng.choice(["bf16", "f16", "f32"]), block=rng.choice([8, 16, 16, 24, 32, 64, 128]),
                     layout=rng.choice(["head", "token"]), bits=bits, **_rotary_draw(rng))
            if sum(_new_lens(c)) == 0 or c["q_heads"] > 128:
                continue
        else:
            kv, group = rng.choice([1, 2, 4, 8, 8, 16, 32]), rng.choice([1, 2, 4, 4, 7, 8, 8, 16])
            kind = rng.choice(["decode", "drafts", "prompts", "chunk", "mixed"])
            ctx = sorted((_log_int(rng, 1, 131071), _log_int(rng, 1, 131071)))
            q = {"decode": [1, 1], "drafts": sorted((rng.randint(1, 8), rng.randint(1, 8))),
                 "prompts": sorted((_log_int(rng, 9, 2048), _log_int(rng, 9, 2048))),
                 "chunk": [_log_int(rng, 65, 4096)] * 2, "mixed": [1, _log_int(rng, 64, 1024)]}[kind]
            requests = 1 if kind == "chunk" else _log_int(rng, 1, 128)
            c = dict(op=op, requests=requests, q_lo=q[0], q_hi=q[1], ctx_lo=0 if kind == "prompts" else ctx[0],
                     ctx_hi=0 if kind == "prompts" else ctx[1], q_heads=kv * group, kv_heads=kv,
                     dim=rng.choice([64, 128, 128]), dtype=rng.choice(["bf16", "f16"]),
                     block=rng.choice([8, 16, 16, 24, 32, 64, 128]), window=rng.choice([0, 0, 0, 4096, 1000]),
                     layout=rng.choice(["head", "token"]))
            q_max, kv_max = max(_q_lens(c)), max(_q_lens(c)) + max(_ctx_lens(c))
            padded = requests * kv * group * q_max * kv_max * 4 + requests * kv_max * kv * c["dim"] * 8
            if kv * group > 128 or padded > 8e9:
                continue
        if _cost(c) <= most:
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


def _size(c):
    return torch.empty(0, dtype=DTYPES[c["dtype"]]).element_size()


def work(case):
    c = case
    if c["op"] == "rotate":
        rows = c["tokens"] * c["heads"]
        return {"bytes": 2 * rows * c["dim"] * _size(c) + 4 * c["tokens"], "flops": 3 * rows * c["rotary_dim"]}
    if c["op"] == "append":
        n, row = sum(_new_lens(c)), c["dim"] * _size(c)
        # queries in and out, keys and values in, their rows of the cache out, a slot and a position a token
        moved = n * (2 * c["q_heads"] * row + 2 * c["kv_heads"] * (row + (c["dim"] if c["bits"] == 8 else row)) + 8)
        return {"bytes": moved, "flops": 3 * n * (c["q_heads"] + c["kv_heads"]) * c["rotary_dim"]}
    seen = keys = 0
    for q, ctx in zip(_q_lens(c), _ctx_lens(c)):
        w = c["window"] or ctx + q
        keys += min(ctx + q, w + q - 1)
        full = max(0, min(q, w - ctx))  # queries that see everything before them
        seen += full * ctx + full * (full + 1) // 2 + (q - full) * w
    rows = 2 * sum(_q_lens(c)) * c["q_heads"] * c["dim"]
    # a byte an element of K and V, two scales a block and head, a table entry a block
    return {"bytes": 2 * rows + 2 * keys * c["kv_heads"] * c["dim"] + (8 * c["kv_heads"] + 4) * keys // c["block"],
            "flops": 4 * seen * c["q_heads"] * c["dim"]}


# -------------------------------------------------------------------------------------------- inputs

def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _indptr(lens):
    return torch.nn.functional.pad(torch.cumsum(_i32(lens), 0), (1, 0)).to(torch.int32)


def _freqs(c):
    """Radians a position of each pair: powers of the base, left alone, slowed down together, or in bands (fast pairs left
    alone, slow ones slowed down by 8, those between by something between)."""
    out = []
    for i in range(c["rotary_dim"] // 2):
        f = (500000.0 if c["scaling"] == "bands" else 10000.0) ** (-2.0 * i / c["rotary_dim"])
        if c["scaling"] == "linear":
            f /= 4.0
        elif c["scaling"] == "bands":
            turns = 8192.0 * f / (2 * math.pi)  # over the length that the model was trained on
            keep = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
            f = keep * f + (1.0 - keep) * f / 8.0
        out.append(f)
    return out


def _rotary(c):
    f = _freqs(c)
    return dict(freqs=torch.tensor(f, dtype=torch.float64, device=DEV), interleaved=c["interleaved"],
                factor=1.1 if c["scaling"] == "linear" else 1.0,
                # the same as whole numbers of 2^-64 turns, the handle that a program keeps
                turns=torch.tensor([int(x / (2 * math.pi) * 2.0 ** 64) for x in f], dtype=torch.int64, device=DEV))


def _cache(num_blocks, c, dtype):
    """Empty [blocks, block, heads, dim], held token by token or head by head."""
    a, b = (c["block"], c["kv_heads"]) if c["layout"] == "token" else (c["kv_heads"], c["block"])
    t = torch.empty(num_blocks, a, b, c["dim"], dtype=dtype, device=DEV)
    return t if c["layout"] == "token" else t.permute(0, 2, 1, 3)


def _filled(num_blocks, c, g):
    """A cache of codes and its scales, of values whose size changes from block to block and head to head."""
    codes = _cache(num_blocks, c, E4M3)
    scales = torch.empty(num_blocks, c["kv_heads"], device=DEV)
    step = max(1, (1 << 27) // (c["block"] * c["kv_heads"] * c["dim"]))
    for at in range(0, num_blocks, step):  # a part at a time: the largest cache in 32 bits would not fit three times
        n = min(step, num_blocks - at)
        x = torch.randn(n, c["block"], c["kv_heads"], c["dim"], generator=g, device=DEV)
        x *= torch.exp(0.25 * torch.randn(n, 1, c["kv_heads"], 1, generator=g, device=DEV))
        f = _scale_for(x.abs().amax((1, 3)))
        codes[at:at + n].copy_((x / f[:, None, :, None]).to(E4M3))
        scales[at:at + n] = f
    return codes, scales


def _scale_for(largest):
    """2^k with the smallest k for which largest <= 448 * 2^k."""
    m, e = torch.frexp(largest)
    k = e - 9 + (m > MOST / 512).to(e.dtype)
    return torch.where(largest > 0, torch.ldexp(torch.ones_like(largest), k), torch.zeros_like(largest)).clamp(min=LEAST)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    if c["op"] == "rotate":
        x = torch.randn(c["tokens"], c["heads"], c["dim"], generator=g, device=DEV, dtype=DTYPES[c["dtype"]])
        positions = torch.randint(0, c["pos_hi"] + 1, (c["tokens"],), generator=g, device=DEV, dtype=torch.int32)
        return dict(op="rotate", x=x, positions=positions, **_rotary(c))
    if c["op"] == "append":
        dtype, b, new, ctx = DTYPES[c["dtype"]], c["block"], _new_lens(c), _ctx_lens(c)
        n, rows = sum(new), sum(new) + c["padding"]
        # the blocks that new tokens land in, in no order
        page = [[(x + t) // b - x // b for t in range(m)] for x, m in zip(ctx, new)]
        first, count = [], 0
        for p in page:
            first.append(count)
            count += p[-1] + 1 if p else 0
        perm = torch.randperm(count + 8, generator=g, device=DEV, dtype=torch.int32)
        own_page = torch.tensor([f + i for f, p in zip(first, page) for i in p], device=DEV)
        offsets = _i32([(x + t) % b for x, m in zip(ctx, new) for t in range(m)])
        slots = torch.nn.functional.pad(perm[own_page] * b + offsets, (0, c["padding"]), value=-1)
        positions = torch.nn.functional.pad(_i32([x + t for x, m in zip(ctx, new) for t in range(m)]), (0, c["padding"]))
        qkv = torch.randn(rows, c["q_heads"] + 2 * c["kv_heads"], c["dim"], generator=g, device=DEV, dtype=dtype)
        q, k, v = qkv.split([c["q_heads"], c["kv_heads"], c["kv_heads"]], 1)
        s = dict(op="append", q=q, k=k, v=v, slots=slots, positions=positions, tokens=n, block=b, k_scales=None, v_scales=None,
                 begins=torch.cumsum(torch.tensor([0] + [m for m in new if m], device=DEV), 0)[:-1], **_rotary(c))
        if c["bits"] == 8:
            s["k_cache"], s["k_scales"] = _filled(count + 8, c, g)
            s["v_cache"], s["v_scales"] = _filled(count + 8, c, g)
            # requests whose earlier rows are smaller than the new ones: their blocks' scales grow
            for name in ("k_scales", "v_scales"):
                s[name] *= torch.where(torch.rand(s[name].shape, generator=g, device=DEV) < 0.3, 0.25, 1.0)
        else:
            for name in ("k_cache", "v_cache"):
                s[name] = _cache(count + 8, c, dtype)
                s[name].copy_(torch.randn(s[name].shape, generator=g, device=DEV, dtype=dtype))
        return s
    b, q_lens = c["block"], _q_lens(c)
    kv_lens = [q + x for q, x in zip(q_lens, _ctx_lens(c))]
    held = _i32([-(-n // b) for n in kv_lens])
    num_blocks = sum(-(-n // b) for n in kv_lens) + 8
    # distinct blocks for every request, in no order, with -1 past a request's own
    perm = torch.randperm(num_blocks, generator=g, device=DEV, dtype=torch.int32)
    j = torch.arange(int(max(kv_lens) // b) + 2, device=DEV)
    at = ((torch.cumsum(held, 0) - held)[:, None] + j).clamp(max=num_blocks - 1)
    tables = torch.where(j < held[:, None], perm[at], torch.full_like(perm[at], -1))
    # scores with a standard deviation of two: attention that is neither flat nor on one key
    q = 2 * torch.randn(sum(q_lens), c["q_heads"], c["dim"], generator=g, device=DEV, dtype=DTYPES[c["dtype"]])
    k_cache, k_scales = _filled(num_blocks, c, g)
    v_cache, v_scales = _filled(num_blocks, c, g)
    return dict(op="attend", q=q, k_cache=k_cache, v_cache=v_cache, k_scales=k_scales, v_scales=v_scales, tables=tables,
                kv_lens=_i32(kv_lens), q_indptr=_indptr(q_lens), max_q_len=max(q_lens), max_kv_len=max(kv_lens),
                window=c["window"], scale=c["dim"] ** -0.5,
                workspace=torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8, device=DEV))


# ---------------------------------------------------------------------------------------- plain forms

def _turned(s, x, positions):
    """x rotated, in 32 bits; angles in 64."""
    angle = positions.double()[:, None, None] * s["freqs"]
    cos, sin = torch.cos(angle).float() * s["factor"], torch.sin(angle).float() * s["factor"]
    n = 2 * s["freqs"].shape[0]
    x = x.float()
    if s["interleaved"]:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :n // 2], x[..., n // 2:n]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., n:]], -1)


def _plain_rotate(s):
    return _turned(s, s["x"], s["positions"]).to(s["x"].dtype)


def _plain_append(s):
    n, b, slots = s["tokens"], s["block"], s["slots"][:s["tokens"]].long()  # the padding at the end has no slot
    q = _turned(s, s["q"], s["positions"]).to(s["q"].dtype)
    k = _turned(s, s["k"], s["positions"])[:n]
    block, off = slots // b, slots % b
    if s["k_scales"] is None:
        s["k_cache"][block, off] = k.to(s["k"].dtype)
        s["v_cache"][block, off] = s["v"][:n]
        return dict(q=q, k_cache=s["k_cache"], v_cache=s["v_cache"])
    for x, codes, scales in ((k, s["k_cache"], s["k_scales"]), (s["v"][:n].float(), s["v_cache"], s["v_scales"])):
        largest = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
        need = torch.zeros_like(scales).index_reduce_(0, block, largest, "amax")
        need = _scale_for(need)
        # the block that each request's first new row lies in may hold rows of earlier calls
        begun, before = block[s["begins"]], off[s["begins"]]
        old = scales[begun]
        fresh = (before == 0)[:, None]
        kept = torch.where(fresh, need[begun], torch.maximum(old, need[begun]))
        scales[block] = need[block]
        scales[begun] = kept
        was = codes[begun].float()
        follows = (torch.arange(b, device=DEV) < before[:, None])[..., None, None]
        now = (was * (old / kept)[:, None, :, None]).to(E4M3)
        codes[begun] = torch.where(follows, now.view(torch.uint8), codes[begun].view(torch.uint8)).view(E4M3)
        codes[block, off] = (x / scales[block][..., None]).clamp(-MOST, MOST).to(E4M3)
    return dict(q=q, k_cache=s["k_cache"], v_cache=s["v_cache"], k_scales=s["k_scales"], v_scales=s["v_scales"])


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
    k = (s["k_cache"][block, j % b].float() * s["k_scales"][block][..., None]).permute(0, 2, 3, 1)
    v = (s["v_cache"][block, j % b].float() * s["v_scales"][block][..., None]).permute(0, 2, 1, 3)
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


def run(state):
    s = state
    if not own:
        return {"rotate": _plain_rotate, "append": _plain_append, "attend": _plain_attend}[s["op"]](s)
    from multi_lora_b200 import paged_kv, rotary

    if s["op"] == "attend":
        return paged_kv.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["kv_lens"], s["q_indptr"],
                                        max_q_len=s["max_q_len"], scale=s["scale"], window=s["window"],
                                        k_scales=s["k_scales"], v_scales=s["v_scales"], workspace=s["workspace"])
    angles = rotary.RotaryPositions(s["turns"], interleaved=s["interleaved"], factor=s["factor"])
    if s["op"] == "rotate":
        return rotary.rotate(s["x"], s["positions"], angles)
    q = paged_kv.append_paged_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], positions=s["positions"],
                                 rotary=angles, q=s["q"], k_scales=s["k_scales"], v_scales=s["v_scales"])
    out = dict(q=q, k_cache=s["k_cache"], v_cache=s["v_cache"])
    return out if s["k_scales"] is None else dict(out, k_scales=s["k_scales"], v_scales=s["v_scales"])


# ------------------------------------------------------------------------------- definitions in 64 bits

def exact(case, seed):
    c = case
    s = prepare(c, seed)
    return {"rotate": _exact_rotate, "append": _exact_append, "attend": _exact_attend}[c["op"]](c, s)


def _exact_turn(c, s, x, positions):
    """Each pair as a complex number times e^(i position f)."""
    f = torch.tensor(_freqs(c), dtype=torch.float64, device=DEV)
    phase = torch.polar(torch.full_like(f, s["factor"]).expand(len(positions), -1), positions[:, None] * f)[:, None]
    half, out = len(f), x.double()
    even = torch.arange(half, device=DEV) * (2 if c["interleaved"] else 1)
    odd = even + (1 if c["interleaved"] else half)
    z = torch.complex(out[..., even], out[..., odd]) * phase
    out[..., even], out[..., odd] = z.real, z.imag
    return out


def _exact_rotate(c, s):
    return _exact_turn(c, s, s["x"], s["positions"])


def _exact_append(c, s):
    n, b = s["tokens"], c["block"]
    at = s["slots"][:n].long()
    out = dict(q=_exact_turn(c, s, s["q"], s["positions"]))
    new = dict(k=_exact_turn(c, s, s["k"], s["positions"])[:n], v=s["v"][:n].double())
    for side, x in new.items():
        cache = s[side + "_cache"].double()
        if c["bits"] == 8:
            # each block as its own list of new rows: their range of offsets, and the largest magnitude a head
            scales = s[side + "_scales"].double()
            first = torch.full((cache.shape[0],), b, device=DEV).scatter_reduce_(0, at // b, at % b, "amin")
            top = torch.zeros_like(scales)
            top.scatter_reduce_(0, (at // b)[:, None].expand(-1, c["kv_heads"]), x.abs().amax(-1), "amax")
            need = torch.exp2(torch.ceil(torch.log2(top / MOST))).clamp(min=LEAST)
            now = torch.where((first == 0)[:, None], need, torch.maximum(scales, need))
            now = torch.where((first == b)[:, None], scales, now)
            stays = (torch.arange(b, device=DEV) < first[:, None])[..., None, None] & (first < b)[:, None, None, None]
            cache = torch.where(stays, cache * (scales / now)[:, None, :, None], cache)
            x = x / now[at // b][..., None]
            out[side + "_scales"] = now
        cache.index_put_((at // b, at % b), x)
        out[side + "_cache"] = cache
    return out


def _exact_attend(c, s):
    group, b = c["q_heads"] // c["kv_heads"], c["block"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    at = 0
    for i, (n, ctx) in enumerate(zip(_q_lens(c), _ctx_lens(c))):
        key = torch.arange(ctx + n, device=DEV)
        page = s["tables"][i].long()[key // b]
        for h in range(c["kv_heads"]):
            k, v = (s[side + "_cache"][page, key % b, h].double() * s[side + "_scales"][page, h].double()[:, None] for side in "kv")
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
