"""The paged serving step in plain Python and 64-bit numpy, from its definitions.

Only tests use it. Every function takes and returns host values; nothing here
shares code with the library.
"""

from __future__ import annotations

import numpy as np


def plan(ctx, new, held, free, head, tables, block, max_tokens):
    """Blocks, slots and positions of a step, one request and one token at a time."""
    tables = [list(row) for row in tables]
    held, width = list(held), len(tables[0]) if len(tables) else 0
    q_indptr, kv_lens, positions, slots = [0], [], [], []
    for i, (c, n) in enumerate(zip(ctx, new)):
        while held[i] < width and held[i] * block < c + n and head < len(free):
            tables[i][held[i]] = free[head]
            held[i] += 1
            head += 1
        for p in range(c, c + n):
            positions.append(p)
            slots.append(tables[i][p // block] * block + p % block if p // block < held[i] else -1)
        q_indptr.append(q_indptr[-1] + n)
        kv_lens.append(c + n)
    pad = max_tokens - len(slots)
    return dict(q_indptr=q_indptr, kv_lens=kv_lens, held=held, head=head, tables=tables,
                positions=positions + [0] * pad, slots=slots + [-1] * pad)


def attention(q, k_cache, v_cache, tables, kv_lens, q_indptr, scale, window=0):
    """(out, mean |v| under the probabilities, largest sum |q_d k_d| scale, keys seen) per query row, float64.

    q [T, Hq, D], caches [num_blocks, block, Hkv, D]; blocks outside the cache count as zeros."""
    q, k_cache, v_cache = (np.asarray(t, np.float64) for t in (q, k_cache, v_cache))
    tokens, heads, dim = q.shape
    num_blocks, block, kv_heads, _ = k_cache.shape
    out, mean = np.zeros(q.shape), np.zeros(q.shape)
    spread, seen = np.zeros((tokens, heads, 1)), np.zeros((tokens, heads, 1))
    for i in range(len(kv_lens)):
        t0, t1 = q_indptr[i], q_indptr[i + 1]
        for t in range(t0, t1):
            pos = kv_lens[i] - (t1 - t0) + (t - t0)
            first = max(0, pos - window + 1) if window else 0
            if pos < first:
                continue
            keys = np.arange(first, pos + 1)
            b = np.asarray(tables[i])[keys // block]
            ok = (b >= 0) & (b < num_blocks)
            at = np.where(ok, b, 0)
            for g in range(kv_heads):
                k = np.where(ok[:, None], k_cache[at, keys % block, g], 0.0)
                v = np.where(ok[:, None], v_cache[at, keys % block, g], 0.0)
                rows = slice(g * (heads // kv_heads), (g + 1) * (heads // kv_heads))
                s = scale * q[t, rows] @ k.T
                p = np.exp(s - s.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                out[t, rows], mean[t, rows] = p @ v, p @ np.abs(v)
                spread[t, rows, 0] = scale * (np.abs(q[t, rows]) @ np.abs(k).T).max(1)
                seen[t, rows, 0] = len(keys)
    return out, mean, spread, seen


def rotate(x, positions, radians, interleaved=False, factor=1.0):
    """x [T, H, D] with pair i of row t turned by positions[t] * radians[i], each pair as a complex number."""
    out = np.array(x, np.float64)
    for i, f in enumerate(radians):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + len(radians))
        turn = factor * np.exp(1j * np.asarray(positions, np.float64) * f)[:, None]
        z = (out[..., a] + 1j * out[..., b]) * turn
        out[..., a], out[..., b] = z.real, z.imag
    return out


def round_e4m3(x):
    """The nearest of e4m3's values (even on a tie): 1.mmm * 2^e for e from -6 to 8, multiples of 2^-9 below; at most 448."""
    x = np.asarray(x, np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.clip(np.floor(np.log2(np.abs(x))), -6, 8)
    step = 2.0 ** (np.where(np.isfinite(e), e, 8) - 3)
    return np.where(np.isnan(x), np.nan, np.clip(np.round(np.clip(x, -448, 448) / step) * step, -448, 448))


def append_codes(values, scales, rows, slots, block):
    """New rows [T, H, D] into a cache of codes: (code values, scales, codes before they are rounded), a block at a time.

    values [num_blocks, block, H, D] are what the codes stand for over their scale, scales [num_blocks, H]."""
    values, scales, rows = (np.array(t, np.float64) for t in (values, scales, rows))
    exact = values.copy()
    slots = np.asarray(slots)
    for b in np.unique(slots[slots >= 0] // block):
        mine = np.flatnonzero((slots >= 0) & (slots // block == b))
        first = int((slots[mine] % block).min())
        size = np.where(np.isfinite(rows[mine]), np.abs(rows[mine]), 0.0).max((0, 2))
        for h, most in enumerate(size):
            k = -100
            while 448.0 * 2.0 ** k < most:
                k += 1
            old, f = scales[b, h], 2.0 ** k
            if first > 0:
                f = max(f, old)
                values[b, :first, h] = round_e4m3(values[b, :first, h] * (old / f))
                exact[b, :first, h] = values[b, :first, h]
            scales[b, h] = f
            exact[b, slots[mine] % block, h] = rows[mine, h] / f
            values[b, slots[mine] % block, h] = round_e4m3(rows[mine, h] / f)
    return values, scales, exact


def verify(target, draft, draft_tokens, row_indptr, accept_u, sample_u):
    """Emitted tokens (-1 behind the last) and their number, with Python's whole numbers for the 40-bit weights.

    target float32 [rows, V], draft float32 [R, K, V] or None."""
    requests, most = np.asarray(draft_tokens).shape
    tokens, emitted = [], []
    for i in range(requests):
        r0, n = row_indptr[i], row_indptr[i + 1] - row_indptr[i] - 1
        if n < 0:
            tokens.append([-1] * (most + 1))
            emitted.append(0)
            continue
        kept = 0
        while kept < n:
            x = int(draft_tokens[i][kept])
            if not 0 <= x < target.shape[1]:
                break
            qx = np.float32(1.0) if draft is None else np.float32(draft[i, kept, x])
            if not np.float32(accept_u[i][kept]) * qx < np.float32(target[r0 + kept, x]):
                break
            kept += 1
        p = np.asarray(target[r0 + kept], np.float32)
        left = p.copy()
        if kept < n:
            if draft is None:
                if 0 <= draft_tokens[i][kept] < target.shape[1]:
                    left[int(draft_tokens[i][kept])] = 0
            else:
                left = p - np.asarray(draft[i, kept], np.float32)

        def weights(x):
            x = np.where(x > 0, np.minimum(x, np.float32(1.0)), np.float32(0.0))  # not positive, NaN: nothing
            return np.floor(x.astype(np.float64) * 2.0 ** 40).astype(np.int64)

        w = weights(left)
        if w.sum() == 0:
            w = weights(p)
        total = int(w.sum())
        place = total * min(max(int(float(sample_u[i]) * 2 ** 24), 0), 2 ** 24 - 1) >> 24
        drawn = int(np.searchsorted(np.cumsum(w), place, side="right")) if total else -1
        row = [int(x) for x in draft_tokens[i][:kept]] + [drawn]
        tokens.append(row + [-1] * (most + 1 - len(row)))
        emitted.append(kept + 1)
    return np.array(tokens), np.array(emitted)
