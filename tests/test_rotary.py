"""Rotary positions and the 8-bit cache on the host: frequencies, the oracle's own sense, refusals and launches (no GPU needed)."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from fake_cudart import FakeLib
from test_paged import cache

from multi_lora_b200 import _native, paged_kv, rotary
from oracle import paged_oracle as O

CPU = torch.device("cpu")
E4M3 = 3


def radians(r):
    """The frequencies that the whole numbers stand for."""
    return [t / 2.0 ** 64 * 2 * math.pi for t in r.turns.tolist()]


def test_frequencies_are_powers_of_the_base():
    r = rotary.RotaryPositions.new(128, CPU, base=500000.0, interleaved=True)
    np.testing.assert_allclose(radians(r), [500000.0 ** (-2 * i / 128) for i in range(64)],
                               rtol=1e-15, atol=2 * math.pi * 2.0 ** -64)  # less than one whole number is cut off
    assert r.interleaved and r.factor == 1.0 and r.turns.dtype == torch.int64
    assert rotary.RotaryPositions.new(2, CPU).turns.tolist() == [int(2.0 ** 64 / (2 * math.pi))]


def test_any_frequency_is_taken_modulo_a_turn():
    r = rotary.RotaryPositions.from_frequencies([0.0, 4.0, -1.0, 2 * math.pi * 3.25], CPU, factor=0.5)
    np.testing.assert_allclose([math.cos(f) for f in radians(r)], [1, math.cos(4.0), math.cos(1.0), 0], atol=1e-14)
    np.testing.assert_allclose([math.sin(f) for f in radians(r)], [0, math.sin(4.0), -math.sin(1.0), 1], atol=1e-14)
    assert all(-2 ** 63 <= t < 2 ** 63 for t in r.turns.tolist()) and r.factor == 0.5


@pytest.mark.parametrize("scaling", [
    {"rope_type": "linear", "factor": 4.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 8192},
    {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096},
    {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 2048, "attention_factor": 0.9},
    {"rope_type": "default"},
])
def test_scaled_frequencies_are_the_model_library_s(scaling):
    """The configuration's own reading of them, which is in fp32."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    kind = scaling.get("rope_type", scaling.get("type"))
    if kind == "default":
        want, factor = torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)]), 1.0
    else:
        config = LlamaConfig(hidden_size=256, num_attention_heads=4, head_dim=64, max_position_embeddings=32768,
                             rope_parameters={"rope_theta": 10000.0, **scaling, "rope_type": kind})
        want, factor = ROPE_INIT_FUNCTIONS[kind](config, CPU)
    r = rotary.RotaryPositions.new(64, CPU, scaling=scaling)
    # fp32 frequencies, blends and powers: a few units of 2^-24
    np.testing.assert_allclose(radians(r), want.double().numpy(), rtol=2.0 ** -20)
    assert r.factor == pytest.approx(factor, rel=1e-6)


def test_refused_frequencies():
    for bad in (0, 3, -2):
        with pytest.raises(ValueError, match="rotary_dim"):
            rotary.RotaryPositions.new(bad, CPU)
    with pytest.raises(ValueError, match="rope_type"):
        rotary.RotaryPositions.new(8, CPU, scaling={"rope_type": "cubic"})
    with pytest.raises(ValueError, match="frequency"):
        rotary.RotaryPositions.from_frequencies([math.inf], CPU)


def test_oracle_rounds_like_the_type():
    x = np.concatenate([np.linspace(-500, 500, 4001), np.linspace(-0.05, 0.05, 4001), [0.0, 2.0 ** -10, 3 * 2.0 ** -10, np.nan]])
    want = torch.tensor(x).clamp(-448, 448).float().to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(O.round_e4m3(x.astype(np.float32)), want)


def test_oracle_append_by_hand():
    values, scales = np.zeros((2, 4, 1, 2)), np.full((2, 1), 0.25)
    values[1, 0, 0] = [100, 3]
    new, f, exact = O.append_codes(values, scales, [[[448.0, -1.0]], [[1.0, 449.0]]], [5, 6], 4)
    assert f.tolist() == [[0.25], [2.0]]
    assert new[1, :3, 0].tolist() == [[12.0, 0.375], [224.0, -0.5], [0.5, 224.0]] and exact[1, 2, 0, 1] == 224.5
    new, f, _ = O.append_codes(values, scales, [[[0.0, 7.0]]], [4], 4)  # a block that begins again
    assert f[1, 0] == 2.0 ** -6 and new[1, 0, 0].tolist() == [0, 448]


def test_oracle_rotation_turns_pairs():
    x = np.arange(1.0, 7.0).reshape(1, 1, 6)
    out = O.rotate(x, [3], [math.pi / 6, 0.0], factor=2.0)
    np.testing.assert_allclose(out[0, 0], [-6, 4, 2, 8, 5, 6], atol=1e-12)
    out = O.rotate(x, [3], [math.pi / 6], interleaved=True)
    np.testing.assert_allclose(out[0, 0], [-2, 1, 3, 4, 5, 6], atol=1e-12)


# ------------------------------------------------------------------------------------------- refusals

def rot(**kw):
    r = _native.RotaryT()
    r.turns, r.pairs, r.interleaved, r.factor = 256, 32, 0, 1.0
    for name, value in kw.items():
        setattr(r, name, value)
    return r


def scales(**kw):
    s = _native.PagedScalesT()
    s.k = s.v = 256
    s.k_block_stride = s.v_block_stride = 2
    s.k_head_stride = s.v_head_stride = 1
    for name, value in kw.items():
        setattr(s, name, value)
    return s


def rotate(lib, r=rot(), **kw):
    a = dict(x=256, xt=128, xh=64, tokens=3, heads=2, dim=64, pos=256, out=4096, ot=128, oh=64, dtype=0)
    a.update(kw)
    return lib.mlora_rotate(a["x"], a["xt"], a["xh"], a["tokens"], a["heads"], a["dim"], a["pos"],
                            None if r is None else ctypes.byref(r), a["out"], a["ot"], a["oh"], a["dtype"], None)


def append(lib, c=None, s=None, r=rot(), **kw):
    a = dict(q=256, qt=256, qh=64, heads=4, out=4096, ot=256, oh=64, k=256, kt=128, kh=64, v=256, vt=128, vh=64, tokens=3,
             dtype=0, pos=256, slots=256)
    a.update(kw)
    return lib.mlora_append_paged_kv(a["q"], a["qt"], a["qh"], a["heads"], a["out"], a["ot"], a["oh"], a["k"], a["kt"],
                                     a["kh"], a["v"], a["vt"], a["vh"], a["tokens"], a["dtype"], ctypes.byref(c or cache()),
                                     None if s is None else ctypes.byref(s), None if r is None else ctypes.byref(r),
                                     a["pos"], a["slots"], None, None)


def attend(lib, c=None, s=scales(), **kw):
    a = dict(q=256, qt=256, qh=64, tokens=2, heads=4, dtype=0, tables=256, rows=4, width=4, kv=256, ind=256, r=2, most=1,
             scale=1.0, window=0, out=256, ot=256, oh=64, ws=256, wb=paged_kv.ATTENTION_WORKSPACE_BYTES)
    a.update(kw)
    return lib.mlora_paged_attention_8bit(a["q"], a["qt"], a["qh"], a["tokens"], a["heads"], a["dtype"],
                                          ctypes.byref(c or cache(dtype=E4M3)), None if s is None else ctypes.byref(s),
                                          a["tables"], a["rows"], a["width"], a["kv"], a["ind"], a["r"], a["most"],
                                          a["scale"], a["window"], a["out"], a["ot"], a["oh"], a["ws"], a["wb"], None, None)


@pytest.mark.parametrize("r, kw, code", [
    (rot(pairs=0), {}, -1), (rot(pairs=33), {}, -1), (rot(turns=None), {}, -1), (None, {}, -1), (rot(), dict(dtype=3), -2),
    (rot(), dict(dtype=7), -2), (rot(), dict(dim=0), -1), (rot(), dict(dim=520), -1), (rot(), dict(tokens=-1), -1),
    (rot(), dict(heads=-1), -1), (rot(), dict(tokens=2 ** 31), -1), (rot(), dict(xt=-1), -1), (rot(), dict(oh=63), -1),
    (rot(), dict(ot=63), -1), (rot(), dict(x=None), -1), (rot(), dict(out=None), -1), (rot(), dict(pos=None), -1),
])
def test_rotate_refusals(r, kw, code):
    lib = _native.capi()
    assert rotate(lib, r, **kw) == code and lib.mlora_last_error()


@pytest.mark.parametrize("c, s, r, kw, code", [
    ({}, None, rot(), dict(dtype=1), -1), (dict(dtype=E4M3), None, rot(), {}, -2), ({}, scales(), rot(), {}, -2),
    (dict(dtype=E4M3), scales(k=None), rot(), {}, -1), (dict(dtype=E4M3), scales(v_head_stride=-1), rot(), {}, -1),
    (dict(dtype=E4M3, block_size=2049), scales(), rot(), {}, -1), ({}, None, None, {}, -1), ({}, None, rot(pairs=40), {}, -1),
    ({}, None, rot(), dict(pos=None), -1), ({}, None, rot(), dict(slots=None), -1), ({}, None, rot(), dict(k=None), -1),
    ({}, None, rot(), dict(q=None), -1), ({}, None, rot(), dict(out=None), -1), ({}, None, rot(), dict(oh=8), -1),
    ({}, None, rot(), dict(tokens=-1), -1), ({}, None, rot(), dict(tokens=2 ** 30), -1), ({}, None, rot(), dict(heads=-1), -1),
    ({}, None, rot(), dict(heads=2 ** 31 - 1), -1), ({}, None, rot(), dict(kt=-1), -1), (dict(head_dim=520), None, rot(), {}, -1),
    (dict(k=None), None, rot(), {}, -1), ({}, None, rot(), dict(dtype=9), -2),
])
def test_append_refusals(c, s, r, kw, code):
    lib = _native.capi()
    assert append(lib, cache(**c), s, r, **kw) == code and lib.mlora_last_error()


@pytest.mark.parametrize("c, s, kw, code", [
    (dict(dtype=0), scales(), {}, -2), (dict(dtype=E4M3), None, {}, -1), (dict(dtype=E4M3), scales(v=None), {}, -1),
    (dict(dtype=E4M3), scales(k_block_stride=-2), {}, -1), (dict(dtype=E4M3), scales(), dict(dtype=3), -2),
    (dict(dtype=E4M3, head_dim=60), scales(), {}, -1), (dict(dtype=E4M3), scales(), dict(heads=5), -1),
    (dict(dtype=E4M3), scales(), dict(window=-1), -1), (dict(dtype=E4M3), scales(), dict(wb=100), -1),
    (dict(dtype=E4M3), scales(), dict(q=None), -1), (dict(dtype=E4M3), scales(), dict(kv=None), -1),
])
def test_attention_refusals(c, s, kw, code):
    lib = _native.capi()
    assert attend(lib, cache(**c), s, **kw) == code and lib.mlora_last_error()


def test_the_other_entry_points_refuse_codes():
    lib = _native.capi()
    c = cache(dtype=E4M3)
    assert lib.mlora_write_paged_kv(256, 128, 64, 256, 128, 64, 3, ctypes.byref(c), 256, None, None) == -2
    assert lib.mlora_paged_attention(256, 256, 64, 2, 4, ctypes.byref(c), 256, 4, 4, 256, 256, 2, 1, 1.0, 0, 256, 256, 64, 256,
                                     paged_kv.ATTENTION_WORKSPACE_BYTES, None, None) == -2


def test_empty_calls_touch_nothing():
    lib = _native.capi()
    assert rotate(lib, tokens=0, x=None, out=None, pos=None) == 0 and rotate(lib, heads=0, x=None, out=None) == 0
    assert append(lib, tokens=0, q=None, out=None, k=None, v=None, slots=None) == 0
    assert attend(lib, tokens=0, q=None, out=None) == 0


def test_cpu_tensors_are_refused():
    z = torch.zeros(1)
    r = rotary.RotaryPositions.new(2, CPU)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary.rotate(z, z, r)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_kv.append_paged_kv(z, z, z, z, z)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_kv.paged_attention(z, z, z, z, z, z, max_q_len=1, workspace=z, k_scales=z, v_scales=z)


def test_a_cache_of_codes_has_scales():
    kw = dict(layers=2, num_blocks=4, block_size=4, kv_heads=3, head_dim=8, max_requests=2, max_blocks=2, device=CPU)
    c = paged_kv.PagedKVCache(dtype=torch.float8_e4m3fn, **kw)
    k, v = c.scales(1)
    assert k.shape == v.shape == (4, 3) and k.dtype == torch.float32 and c.layer(1)[0].dtype == torch.float8_e4m3fn
    assert k.data_ptr() != v.data_ptr() and paged_kv.PagedKVCache(dtype=torch.float32, **kw).scales(0) == (None, None)


# ------------------------------------------------------------------------------------------- launches

@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return FakeLib(tmp_path_factory.mktemp("fake"))


@pytest.mark.parametrize("tokens", [1, 7, 512, 4352, 100000])
@pytest.mark.parametrize("block", [1, 16, 24, 2048])
@pytest.mark.parametrize("dim, pairs", [(64, 32), (128, 16), (5, 2), (512, 256), (72, 36)])
@pytest.mark.parametrize("codes", [False, True])
def test_every_append_launch_has_blocks(fake, tokens, block, dim, pairs, codes):
    fake.reset()
    c = cache(head_dim=dim, block_size=block, dtype=E4M3 if codes else 0, k=4096, v=4096)
    assert append(fake.c, c, scales() if codes else None, rot(pairs=pairs), tokens=tokens, oh=dim, ot=4 * dim) == 0, fake.error()
    (launch,) = fake.launches()
    assert launch.result == 0 and min(launch.grid) > 0 and launch.smem <= (160 if codes else 48) * 1024


@pytest.mark.parametrize("call", [
    lambda f: append(f.c, cache(dtype=E4M3, k=4096, v=4096), scales()),
    lambda f: attend(f.c, cache(dtype=E4M3, k=4096, v=4096), scales(k=4096, v=4096)),
    lambda f: attend(f.c, cache(dtype=E4M3, k=4096, v=4096), scales(k=4096, v=4096), rows=400, width=400),
    lambda f: attend(f.c, cache(dtype=E4M3, k=4096, v=4096), scales(k=4096, v=4096), tokens=200, most=100),
], ids=["append", "cluster", "dealt", "chunk"])
def test_every_device_of_a_process(fake, call):
    for dev in (3, 1, 0, 3, 2, 1):
        fake.reset()
        fake.device(dev)
        assert call(fake) == 0, (dev, fake.error())
        assert [x.device for x in fake.launches()] == [dev]
        fake.reset()
        fake.device(dev)
        assert call(fake) == 0 and fake.c.fake_attribute_calls() == 0


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("width", [0, 4, 256, 4000])
@pytest.mark.parametrize("requests, rows, most", [(0, 5, 1), (0, 300, 100), (1, 5, 1), (40, 50, 1), (40, 300, 90)])
def test_every_attention_launch_has_blocks(fake, requests, rows, most, width, dtype):
    fake.reset()
    assert attend(fake.c, cache(dtype=E4M3, k=4096, v=4096), scales(k=4096, v=4096), q=4096, out=4096, tables=4096, kv=4096,
                  ind=4096, ws=4096, r=requests, tokens=rows, most=most, rows=width, width=width, dtype=dtype) == 0, fake.error()
    launches = fake.launches()
    assert len(launches) == 1 and launches[0].result == 0 and min(launches[0].grid) > 0
