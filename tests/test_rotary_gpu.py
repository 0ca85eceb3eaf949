"""Rotary positions, alone and on the way into the paged cache (16, 32 and 8 bits), against oracle/paged_oracle.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_paged_gpu import DTYPES, host, i32, make_cache, status_word

from multi_lora_b200 import paged_kv as P
from multi_lora_b200.rotary import RotaryPositions, rotate
from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}  # half a step, relative
LEAST = {"bf16": 2.0 ** -134, "f16": 2.0 ** -25, "f32": 2.0 ** -150}  # half a step of subnormals


def freqs(pairs, base=10000.0):
    return [base ** (-i / pairs) for i in range(pairs)]


def fp32_error(x, pairs, interleaved, factor):
    """Of a rotated element before it is rounded: angles (2^-23.3: a half turn in fp32), sincospif (2 units), the factor and
    three operations, each relative to the pair's two elements."""
    a = np.abs(host(x))
    out = np.zeros_like(a)
    n = 2 * pairs
    even, odd = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, pairs), slice(pairs, n))
    out[..., even] = out[..., odd] = a[..., even] + a[..., odd]
    return abs(factor) * out * 2.0 ** -21


def assert_rotated(got, x, positions, pairs, dtype, interleaved=False, factor=1.0, radians=None):
    want = O.rotate(host(x), positions.tolist(), radians or freqs(pairs), interleaved, factor)
    bound = fp32_error(x, pairs, interleaved, factor) + HALF[dtype] * np.abs(want) + LEAST[dtype]
    assert (np.abs(host(got) - want) <= bound).all()
    assert torch.equal(got[..., 2 * pairs:], x[..., 2 * pairs:])


CASES = [
    # tokens, heads, dim, pairs, interleaved
    (1, 1, 2, 1, False), (1, 32, 128, 64, False), (64, 32, 128, 64, True), (5, 3, 72, 36, False), (9, 2, 72, 16, True),
    (33, 7, 96, 20, False), (700, 8, 128, 64, False), (17, 5, 7, 3, True), (3, 4, 256, 128, False), (2, 2, 512, 256, True),
    (40, 1, 64, 16, False), (11, 130, 128, 64, False), (2500, 3, 64, 32, True),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tokens, heads, dim, pairs, interleaved", CASES)
def test_rotate_matches_the_oracle(cuda_dev, dtype, tokens, heads, dim, pairs, interleaved):
    g = torch.Generator(device=cuda_dev).manual_seed(tokens)
    x = torch.randn(tokens, heads + 2, dim, generator=g, device=cuda_dev).to(DTYPES[dtype])[:, 1:heads + 1]
    positions = torch.randint(0, 200000, (tokens,), generator=g, device=cuda_dev).to(torch.int32)
    r = RotaryPositions.from_frequencies(freqs(pairs), cuda_dev, interleaved=interleaved, factor=1.25)
    got = rotate(x, positions, r)
    assert_rotated(got, x, positions, pairs, dtype, interleaved, 1.25)
    wide = torch.full((tokens, 2 * heads, dim), 5.0, dtype=x.dtype, device=cuda_dev)
    assert rotate(x, positions, r, out=wide[:, ::2]).data_ptr() == wide.data_ptr()
    assert torch.equal(wide[:, ::2], got) and (wide[:, 1::2] == 5).all()
    whole = x.clone()  # in place, and a row that starts anywhere
    odd = torch.zeros(whole.numel() + 1, dtype=x.dtype, device=cuda_dev)[1:].view(x.shape).copy_(x)
    assert torch.equal(rotate(whole, positions, r, out=whole), got) and torch.equal(rotate(odd, positions, r, out=odd), got)


@pytest.mark.parametrize("at", [0, 1, 2 ** 20, 2 ** 31 - 1, -1, -(2 ** 31)])
def test_positions_far_away_and_negative(cuda_dev, at):
    """Angles are products of whole numbers: what the position is does not matter to their accuracy."""
    x = torch.randn(3, 2, 64, generator=torch.Generator(device=cuda_dev).manual_seed(1), device=cuda_dev)
    r = RotaryPositions.new(64, cuda_dev)
    positions = i32([at] * 3, cuda_dev)
    # the frequencies as the whole numbers have them: a 64-bit float's would be off by 2^31 * 2^-53 radians
    exact = [(t % 2 ** 64) * at % 2 ** 64 / 2.0 ** 64 * 2 * np.pi for t in r.turns.tolist()]
    want = O.rotate(host(x), [1] * 3, exact)
    assert (np.abs(host(rotate(x, positions, r)) - want) <= fp32_error(x, 32, False, 1.0) + HALF["f32"] * np.abs(want)).all()


def test_rotate_of_nothing(cuda_dev):
    r = RotaryPositions.new(8, cuda_dev)
    for shape in ((0, 4, 8), (4, 0, 8)):
        x = torch.zeros(shape, device=cuda_dev)
        assert rotate(x, torch.zeros(shape[0], dtype=torch.int32, device=cuda_dev), r).shape == shape


def test_infinities_and_nan_stay_in_their_pair(cuda_dev):
    x = torch.ones(1, 1, 16, device=cuda_dev)
    x[0, 0, 3], x[0, 0, 5] = float("inf"), float("nan")
    got = rotate(x, i32([1], cuda_dev), RotaryPositions.new(16, cuda_dev))
    assert torch.isfinite(got).flatten().tolist() == [i % 8 not in (3, 5) for i in range(16)]


# ---------------------------------------------------------------------------------------------- append

def step(dev, seed, requests, new, ctx, block, spare=3, shuffle=True):
    """(slots, positions) of requests with `new` tokens behind `ctx`, blocks in no order, a -1 row behind them."""
    rng = np.random.default_rng(seed)
    pages, slots, positions = [], [], []
    for n, c in zip(new, ctx):
        pages.append((n + c % block + block - 1) // block if n else 0)
    order = rng.permutation(sum(pages) + spare) if shuffle else np.arange(sum(pages) + spare)
    first = 0
    for n, c, p in zip(new, ctx, pages):
        for t in range(c, c + n):
            slots.append(int(order[first + t // block - c // block]) * block + t % block)
            positions.append(t)
        first += p
    return slots, positions, sum(pages) + spare


APPENDS = [
    # new tokens, context, q_heads, kv_heads, dim, pairs, block
    ([1], [0], 4, 4, 128, 64, 16), ([1] * 64, [37 * i for i in range(64)], 32, 8, 128, 64, 16),
    ([3, 0, 70, 1, 129], [5, 9, 0, 31, 14], 8, 2, 128, 64, 16), ([40, 7], [0, 100], 6, 3, 72, 36, 24),
    ([200, 130], [3, 127], 2, 1, 64, 16, 128), ([9, 1, 1], [3, 2, 0], 5, 5, 7, 2, 1), ([300], [77], 4, 2, 96, 48, 48),
    ([2] * 300, [i for i in range(300)], 8, 8, 64, 32, 8), ([900], [500], 2, 1, 128, 64, 2048),
    ([5, 4000], [11, 0], 4, 4, 128, 64, 32), ([33, 33], [0, 31], 1, 1, 256, 128, 64),
]


APPEND_IDS = [f"r{len(a[0])}-n{sum(a[0])}-h{a[2]}.{a[3]}-d{a[4]}.{a[5]}-b{a[6]}" for a in APPENDS]


@pytest.mark.parametrize("layout", ["head", "token", "odd"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("new, ctx, q_heads, kv_heads, dim, pairs, block", APPENDS, ids=APPEND_IDS)
def test_append_rotates_and_places(cuda_dev, dtype, new, ctx, q_heads, kv_heads, dim, pairs, block, layout):
    """Bit for bit what a rotation and a cache write of their own give."""
    g = torch.Generator(device=cuda_dev).manual_seed(len(new))
    slots, positions, blocks = step(cuda_dev, 1, len(new), new, ctx, block)
    n = len(slots) + 2
    slots, positions = i32(slots + [-1, -1], cuda_dev), i32(positions + [0, 7], cuda_dev)
    qkv = torch.randn(n, q_heads + 2 * kv_heads, dim, generator=g, device=cuda_dev).to(DTYPES[dtype])
    q, k, v = qkv.split([q_heads, kv_heads, kv_heads], 1)
    r = RotaryPositions.from_frequencies(freqs(pairs), cuda_dev, interleaved=block % 16 != 0, factor=0.75)
    caches = [make_cache(cuda_dev, blocks, block, kv_heads, dim, DTYPES[dtype], layout, fill=7.0) for _ in range(4)]
    status = status_word(cuda_dev)
    got = P.append_paged_kv(k, v, caches[0], caches[1], slots, positions=positions, rotary=r, q=q, status=status)
    assert torch.equal(got, rotate(q, positions, r))
    assert_rotated(got, q, positions, pairs, dtype, r.interleaved, r.factor)
    P.write_paged_kv(rotate(k, positions, r), v, caches[2], caches[3], slots)
    assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])
    plain = [make_cache(cuda_dev, blocks, block, kv_heads, dim, DTYPES[dtype], layout, fill=7.0) for _ in range(4)]
    assert P.append_paged_kv(k, v, plain[0], plain[1], slots, status=status) is None  # without a rotation
    P.write_paged_kv(k, v, plain[2], plain[3], slots)
    assert torch.equal(plain[0], plain[2]) and torch.equal(plain[1], plain[3])
    assert status.item() == 0


def codes_cache(dev, blocks, block, heads, dim, layout, g):
    """Random codes (NaN among them) and scales, 2^-3 to 2^3."""
    raw = torch.randint(0, 256, (blocks, heads, block, dim + (layout == "odd")), generator=g, device=dev, dtype=torch.uint8)
    t = raw.view(E4M3)[..., :dim].transpose(1, 2)
    if layout == "token":
        t = t.contiguous()
    scales = 2.0 ** torch.randint(-9, -2, (heads, blocks), generator=g, device=dev).float().T
    return t, scales if layout == "head" else scales.contiguous()


def assert_codes(cache, scales, before, before_scales, rows, error, slots, block):
    """`error`: of the rows in fp32, 0 where they are not rotated (codes are the oracle's own then)."""
    values, f, exact = O.append_codes(before, before_scales, rows, slots, block)
    got, got_f = host(cache.float()), host(scales)
    if error is None:
        np.testing.assert_array_equal(got_f, f)
        np.testing.assert_array_equal(got, values)
        return
    # a largest magnitude within the error of a power of two may have either scale: none here
    np.testing.assert_array_equal(got_f, f)
    wide = np.zeros_like(exact)
    slots = np.asarray(slots)
    at = slots >= 0
    b, o = slots[at] // block, slots[at] % block
    wide[b, o] = error[at] / f[b][..., None]
    new = np.zeros(exact.shape[:2], bool)
    new[b, o] = True
    np.testing.assert_array_equal(got[~new], values[~new])
    y = exact[new]
    bound = wide[new] * (1 + 2.0 ** -4) + np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10)
    assert np.array_equal(np.isnan(got[new]), np.isnan(y)) and (np.abs(got[new] - y)[~np.isnan(y)] <= bound[~np.isnan(y)]).all()
    assert (got[new] == values[new])[~np.isnan(y)].mean() > 0.999  # all but those next to a border


@pytest.mark.parametrize("layout", ["head", "token", "odd"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("new, ctx, q_heads, kv_heads, dim, pairs, block", APPENDS, ids=APPEND_IDS)
def test_append_of_codes(cuda_dev, dtype, new, ctx, q_heads, kv_heads, dim, pairs, block, layout):
    g = torch.Generator(device=cuda_dev).manual_seed(len(new) + 1)
    slots, positions, blocks = step(cuda_dev, 2, len(new), new, ctx, block)
    n = len(slots) + 3
    slots, positions = slots + [-1] * 3, positions + [0, 7, 9]
    qkv = torch.randn(n, q_heads + 2 * kv_heads, dim, generator=g, device=cuda_dev)
    qkv = (qkv * 2.0 ** torch.randint(-6, 6, (n, 1, 1), generator=g, device=cuda_dev)).to(DTYPES[dtype])
    q, k, v = qkv.split([q_heads, kv_heads, kv_heads], 1)
    r = RotaryPositions.from_frequencies(freqs(pairs), cuda_dev, interleaved=block % 16 != 0, factor=0.75)
    (kc, ks), (vc, vs) = (codes_cache(cuda_dev, blocks, block, kv_heads, dim, layout, g) for _ in range(2))
    before = [host(t.float()) for t in (kc, ks, vc, vs)]
    status = status_word(cuda_dev)
    got = P.append_paged_kv(k, v, kc, vc, i32(slots, cuda_dev), positions=i32(positions, cuda_dev), rotary=r, q=q, k_scales=ks,
                            v_scales=vs, status=status)
    assert status.item() == 0
    assert torch.equal(got, rotate(q, i32(positions, cuda_dev), r))
    assert_codes(vc, vs, before[2], before[3], host(v), None, slots, block)
    rotated = O.rotate(host(k), positions, freqs(pairs), r.interleaved, r.factor)
    assert_codes(kc, ks, before[0], before[1], rotated, fp32_error(k, pairs, r.interleaved, r.factor), slots, block)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_append_of_codes_without_a_rotation(cuda_dev, dtype):
    """Zeros, infinities, NaN, tiny and huge rows; scales that are no powers of two."""
    g = torch.Generator(device=cuda_dev).manual_seed(3)
    block, blocks, heads, dim = 16, 9, 3, 64
    (kc, ks), (vc, vs) = (codes_cache(cuda_dev, blocks, block, heads, dim, "head", g) for _ in range(2))
    ks.mul_(1.37)
    before = [host(t.float()) for t in (kc, ks, vc, vs)]
    k, v = (torch.randn(40, heads, dim, generator=g, device=cuda_dev) for _ in range(2))
    v[0] = 0
    v[1] = 2.0 ** -120
    k[2, 0, 5], k[2, 1, 6], k[2, 2, 7] = float("inf"), float("-inf"), float("nan")
    v[3:20] *= 1e30
    k[21] *= 2.0 ** -40
    k, v = k.to(DTYPES[dtype]), v.to(DTYPES[dtype])
    slots = [16, 32, 57, *range(64, 81), -1, 100, *range(119, 137)]
    P.append_paged_kv(k, v, kc, vc, i32(slots, cuda_dev), k_scales=ks, v_scales=vs)
    for cache, scales, b, f, x in ((kc, ks, before[0], before[1], k), (vc, vs, before[2], before[3], v)):
        values, want_f, _ = O.append_codes(b, f, host(x), slots, block)
        np.testing.assert_allclose(host(scales), want_f, rtol=2.0 ** -24)
        # divisions by scales that are no powers of two are rounded first: next to a border the code may be the other one
        got = host(cache.float())
        near = np.isclose(got, values, rtol=2.0 ** -3 + 2.0 ** -20, atol=2.0 ** -9, equal_nan=True)
        same = (got == values) | (np.isnan(got) & np.isnan(values))
        assert near.all() and same.mean() > 0.999 and (cache is kc or same.all())


def test_append_token_by_token_is_near_the_values(cuda_dev):
    """A block that fills up in 16 calls, scales growing: every code within its half step and a subnormal half step a growth."""
    g = torch.Generator(device=cuda_dev).manual_seed(4)
    kc, vc = (torch.zeros(2, 16, 2, 64, device=cuda_dev).to(E4M3) for _ in range(2))
    ks, vs = (torch.zeros(2, 2, device=cuda_dev) for _ in range(2))
    x = torch.randn(16, 2, 64, generator=g, device=cuda_dev) * torch.logspace(-2, 2, 16, device=cuda_dev)[:, None, None]
    for t in range(16):
        P.append_paged_kv(x[t:t + 1], x[t:t + 1], kc, vc, i32([16 + t], cuda_dev), k_scales=ks, v_scales=vs)
    f = vs[1].double()[:, None]
    got, want = vc[1].double() * f, x.double()
    assert ((got - want).abs() <= 2.0 ** -4 * want.abs() + 16 * 2.0 ** -10 * f).all()
    most = want.abs().amax((0, 2))
    assert ((448 * f[:, 0] >= most) & (224 * f[:, 0] < most)).all() and torch.equal(ks, vs)
    assert (vc[0].float() == 0).all() and (vs[0] == 0).all()


def test_append_reports_slots_past_the_cache(cuda_dev):
    r = RotaryPositions.new(64, cuda_dev)
    k = torch.ones(4, 1, 64, device=cuda_dev)
    for codes in (False, True):
        kc, vc = (torch.ones(2, 16, 1, 64, device=cuda_dev).to(E4M3 if codes else torch.float32) for _ in range(2))
        f = dict(k_scales=torch.ones(2, 1, device=cuda_dev), v_scales=torch.ones(2, 1, device=cuda_dev)) if codes else {}
        status = status_word(cuda_dev)
        P.append_paged_kv(k, k, kc, vc, i32([32, 33, 31, 2 ** 31 - 1], cuda_dev), positions=i32([0] * 4, cuda_dev), rotary=r,
                          status=status, **f)
        scale = f["v_scales"][1, 0].item() if codes else 1.0
        assert (vc.float()[:, :, 0].reshape(32, 64)[:31] == (1 / scale if codes and scale > 1 else 1)).all()
        assert (vc.float()[1, 15] * scale == 1).all()
        with pytest.raises(RuntimeError, match="slot"):
            P.check_status(status)


def test_append_on_another_stream_and_in_a_graph(cuda_dev):
    g = torch.Generator(device=cuda_dev).manual_seed(5)
    new, ctx = [1] * 12 + [40], [7 * i for i in range(12)] + [0]
    slots, positions, blocks = step(cuda_dev, 3, 13, new, ctx, 16)
    slots, positions = i32(slots, cuda_dev), i32(positions, cuda_dev)
    qkv = torch.randn(slots.numel(), 16, 128, generator=g, device=cuda_dev).bfloat16()
    r = RotaryPositions.new(128, cuda_dev)
    start = [codes_cache(cuda_dev, blocks, 16, 4, 128, "head", g) for _ in range(2)]

    def run(out=None, to=None):
        (kc, ks), (vc, vs) = to or [(c.clone(), f.clone()) for c, f in start]
        q = P.append_paged_kv(qkv[:, 8:12], qkv[:, 12:], kc, vc, slots, positions=positions, rotary=r, q=qkv[:, :8], q_out=out,
                              k_scales=ks, v_scales=vs)
        return [q, kc.view(torch.uint8), ks, vc.view(torch.uint8), vs]

    want = run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    to, out = [(c.clone(), f.clone()) for c, f in start], torch.empty_like(want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = run(out, to)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    # a replay with other rows, positions and slots follows them
    qkv.copy_(torch.randn(qkv.shape, generator=g, device=cuda_dev))
    positions.add_(16)
    for (c, f), (c0, f0) in zip(to, start):
        c.view(torch.uint8).copy_(c0.view(torch.uint8))
        f.copy_(f0)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(again, run()))


def test_refusals_of_tensors(cuda_dev):
    r = RotaryPositions.new(64, cuda_dev)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=cuda_dev)
    at = i32([0, 1, 2], cuda_dev)
    for bad, text in [
        (dict(x=x.long()), "dtype"), (dict(x=x[0]), "x must be"), (dict(x=x.transpose(0, 2)), "x must be"),
        (dict(positions=at.long()), "positions"), (dict(positions=at[:2]), "positions"), (dict(positions=at.cpu()), "positions"),
        (dict(out=x.float()), "out"), (dict(out=x[:2]), "out"), (dict(x=x[..., :32]), "pairs"),
        (dict(rotary=RotaryPositions(r.turns.int())), "turns"), (dict(rotary=RotaryPositions(r.turns[::2])), "turns"),
        (dict(rotary=RotaryPositions(r.turns.cpu())), "turns"), (dict(rotary=RotaryPositions(r.turns[:0])), "pairs"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            rotate(**dict(dict(x=x, positions=at, rotary=r), **bad))
    wide = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=cuda_dev)
    with pytest.raises(RuntimeError, match="overlaps"):
        rotate(wide[:, :2], at, r, out=wide[:, ::2])
    kc, codes = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16, device=cuda_dev), torch.zeros(4, 16, 2, 64, device=cuda_dev).to(E4M3)
    f = torch.ones(4, 2, device=cuda_dev)
    good = dict(k=x, v=x, k_cache=kc, v_cache=kc.clone(), slot_map=at, positions=at, rotary=r, q=wide)
    scaled = dict(good, k_cache=codes, v_cache=codes.clone(), k_scales=f, v_scales=f)
    for base, bad, text in [
        (good, dict(k=x.half()), "dtype"), (good, dict(v=x[:2]), "k and v"), (good, dict(rotary=None), "come together"),
        (good, dict(positions=None), "come together"), (good, dict(rotary=None, positions=None), "rotary is missing"),
        (good, dict(q=wide[:2]), "q must be"), (good, dict(q=wide.float()), "dtype"), (good, dict(q=None, q_out=wide), "q_out"),
        (good, dict(q_out=wide[:, :2]), "q_out"), (good, dict(slot_map=at.long()), "slot_map"), (good, dict(k_scales=f), "together"),
        (good, dict(k_scales=f, v_scales=f), "float8"), (good, dict(k_cache=codes, v_cache=codes), "dtype"),
        (scaled, dict(k_scales=f.half()), "scales"), (scaled, dict(v_scales=f[:3]), "scales"), (scaled, dict(v_scales=f.cpu()), "scales"),
        (scaled, dict(k_scales=None, v_scales=None), "dtype"), (scaled, dict(v_cache=kc), "dtype"), (scaled, dict(k=x.long()), "dtype"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            P.append_paged_kv(**dict(base, **bad))


def test_a_graph_that_is_asked_for_is_not_lost_in_silence(cuda_dev):
    """There is no gradient: the queries come back as torch's operators without one give them, the cache stays out of it."""
    r, at = RotaryPositions.new(64, cuda_dev), i32([0, 1, 2], cuda_dev)
    x = torch.randn(3, 6, 64, device=cuda_dev)
    kc, vc = (torch.zeros(4, 16, 2, 64, device=cuda_dev) for _ in range(2))
    want = P.append_paged_kv(x[:, 2:4], x[:, 4:], kc, vc, at, positions=at, rotary=r, q=x[:, :2])
    x.requires_grad_()
    got = P.append_paged_kv(x[:, 2:4], x[:, 4:], kc, vc, at, positions=at, rotary=r, q=x[:, :2])
    assert got.requires_grad and torch.equal(got, want) and not kc.requires_grad and kc.grad_fn is None
    assert rotate(x, at, r).requires_grad
    with torch.no_grad():
        assert not P.append_paged_kv(x[:, 2:4], x[:, 4:], kc, vc, at, positions=at, rotary=r, q=x[:, :2]).requires_grad
