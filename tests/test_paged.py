"""What the paged serving step refuses before any CUDA call, and the oracle's own sense (no GPU needed)."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from multi_lora_b200 import _native, paged_kv, speculative
from oracle import paged_oracle as O


def cache(**kw):
    c = _native.PagedCacheT()
    c.k = c.v = 256
    c.num_blocks, c.block_size, c.kv_heads, c.head_dim, c.dtype = 8, 16, 2, 64, 0
    for side in "kv":
        for name, value in (("block", 16 * 2 * 64), ("slot", 2 * 64), ("head", 64)):
            setattr(c, f"{side}_{name}_stride", value)
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def attend(c=None, **kw):
    a = dict(q=256, qt=256, qh=64, tokens=2, heads=4, tables=256, rows=4, width=4, kv=256, ind=256, r=2, most=1,
             scale=1.0, window=0, out=256, ot=256, oh=64, ws=256, wb=paged_kv.ATTENTION_WORKSPACE_BYTES)
    a.update(kw)
    lib = _native.capi()
    return lib.mlora_paged_attention(a["q"], a["qt"], a["qh"], a["tokens"], a["heads"], ctypes.byref(c or cache()),
                                     a["tables"], a["rows"], a["width"], a["kv"], a["ind"], a["r"], a["most"],
                                     a["scale"], a["window"], a["out"], a["ot"], a["oh"], a["ws"], a["wb"], None, None)


@pytest.mark.parametrize("c, kw, code", [
    (dict(dtype=7), {}, -2), (dict(block_size=0), {}, -1), (dict(kv_heads=0), {}, -1), (dict(head_dim=60), {}, -1),
    (dict(head_dim=264), {}, -1), (dict(num_blocks=2 ** 30), {}, -1), (dict(k=None), {}, -1),
    (dict(v_slot_stride=-1), {}, -1), ({}, dict(heads=5), -1), ({}, dict(heads=0), -1), ({}, dict(tokens=-1), -1),
    ({}, dict(tokens=2 ** 31), -1), ({}, dict(rows=3), -1), ({}, dict(window=-1), -1), ({}, dict(oh=32), -1),
    ({}, dict(ws=None), -1), ({}, dict(wb=1000), -1), ({}, dict(ws=264), -1), ({}, dict(q=None), -1),
    ({}, dict(kv=None), -1), ({}, dict(ind=None), -1), ({}, dict(most=-1), -1), ({}, dict(width=2 ** 30, rows=2 ** 30), -1),
])
def test_attention_argument_validation(c, kw, code):
    assert attend(cache(**c), **kw) == code
    assert _native.capi().mlora_last_error()


def test_empty_calls_touch_nothing():
    lib = _native.capi()
    assert attend(tokens=0, q=None, out=None) == 0
    assert lib.mlora_write_paged_kv(None, 0, 0, None, 0, 0, 0, ctypes.byref(cache()), None, None, None) == 0
    assert lib.mlora_verify_draft(None, 0, 10, 10, None, 0, 0, None, None, 0, 3, None, None, None, None, 0, None,
                                  None) == 0


def test_write_plan_and_verify_argument_validation():
    lib = _native.capi()
    write = lambda c, *a: lib.mlora_write_paged_kv(*a, ctypes.byref(c), 256, None, None)  # noqa: E731
    assert write(cache(dtype=9), 256, 128, 64, 256, 128, 64, 3) == -2
    assert write(cache(), None, 128, 64, 256, 128, 64, 3) == -1
    assert write(cache(), 256, -1, 64, 256, 128, 64, 3) == -1
    assert write(cache(), 256, 128, 64, 256, 128, 64, -3) == -1
    plan = lambda **k: lib.mlora_plan_paged_step(*(k.get(n, d) for n, d in (  # noqa: E731
        ("ctx", 16), ("new", 16), ("held", 16), ("r", 2), ("free", 16), ("nf", 4), ("head", 16), ("tab", 16),
        ("stride", 4), ("width", 4), ("block", 16), ("ind", 16), ("kv", 16), ("ho", 16), ("fo", 16), ("pos", 16),
        ("slot", 16), ("most", 8), ("ticket", 16), ("status", None), ("stream", None))))
    for bad in (dict(r=-1), dict(r=8193), dict(block=0), dict(width=-1), dict(stride=3), dict(nf=-1), dict(most=-1),
                dict(ind=None), dict(ticket=None), dict(head=None), dict(ctx=None), dict(tab=None), dict(free=None),
                dict(pos=None), dict(r=8192, width=2 ** 19, stride=2 ** 19)):
        assert plan(**bad) == -1, bad
    verify = lambda **k: lib.mlora_verify_draft(*(k.get(n, d) for n, d in (  # noqa: E731
        ("t", 16), ("rows", 4), ("v", 10), ("ts", 10), ("d", 16), ("dr", 20), ("ds", 10), ("x", 16), ("ind", 16),
        ("r", 1), ("k", 2), ("au", 16), ("su", 16), ("out", 16), ("n", 16), ("dt", 2), ("st", None), ("s", None))))
    for bad, code in ((dict(dt=5), -2), (dict(v=0), -1), (dict(v=2 ** 22 + 1, ts=2 ** 23, ds=2 ** 23), -1),
                      (dict(ts=9), -1), (dict(ds=9), -1), (dict(k=-1), -1), (dict(t=None), -1), (dict(su=None), -1),
                      (dict(out=None), -1), (dict(x=None), -1), (dict(r=-1), -1)):
        assert verify(**bad) == code, bad


def test_more_refusals():
    assert attend(ot=32) == -1  # rows of the output that overlap
    assert attend(tokens=1, ot=0, r=0, most=0, oh=8) == -1
    lib = _native.capi()
    plan = lambda r, most: lib.mlora_plan_paged_step(16, 16, 16, r, 16, 4, 16, 16, 4, 4, 16, 16, 16, 16, 16, 16, 16,  # noqa: E731
                                                     most, 16, None, None)
    assert plan(8192, 2 ** 19) == -1 and b"32 bits" in lib.mlora_last_error()


def test_cpu_tensors_are_refused():
    z = torch.zeros(1)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_kv.write_paged_kv(z, z, z, z, z)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_kv.paged_attention(z, z, z, z, z, z, max_q_len=1, workspace=z)
    with pytest.raises(RuntimeError, match="CUDA"):
        speculative.verify_draft(z, None, z, z, z, z)
    with pytest.raises(ValueError):
        paged_kv.PagedKVCache(layers=0, num_blocks=1, block_size=1, kv_heads=1, head_dim=8, max_requests=1,
                              max_blocks=1, dtype=torch.float32, device=torch.device("cpu"))


def test_workspace_size_is_the_library_s():
    assert _native.capi().mlora_paged_attention_workspace_bytes() == paged_kv.ATTENTION_WORKSPACE_BYTES


def test_oracle_plan_by_hand():
    got = O.plan([3, 0, 8], [2, 0, 1], [1, 0, 2], [9, 8, 7], 0, [[5, -1], [-1, -1], [3, 4]], 4, 5)
    assert got["tables"] == [[5, 9], [-1, -1], [3, 4]] and got["held"] == [2, 0, 2] and got["head"] == 1
    assert got["slots"] == [23, 36, -1, -1, -1] and got["positions"] == [3, 4, 8, 0, 0]
    assert got["q_indptr"] == [0, 2, 2, 3]


def test_oracle_attention_is_a_softmax_over_what_is_seen():
    rng = np.random.default_rng(0)
    k, v, q = rng.standard_normal((4, 2, 1, 8)), rng.standard_normal((4, 2, 1, 8)), rng.standard_normal((3, 2, 8))
    out, *_ = O.attention(q, k, v, [[2, 0, 3]], [5], [0, 3], 0.5, window=3)
    kk, vv = k[[2, 0, 3], :, 0].reshape(6, 8), v[[2, 0, 3], :, 0].reshape(6, 8)
    for t, pos in enumerate((2, 3, 4)):
        w = np.exp(0.5 * kk[pos - 2:pos + 1] @ q[t, 1])
        np.testing.assert_allclose(out[t, 1], w @ vv[pos - 2:pos + 1] / w.sum(), rtol=1e-12)
