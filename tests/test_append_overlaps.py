"""What an append or a rotation writes has a place of its own: refusals of scales and rows that share memory (no GPU needed)."""

from __future__ import annotations

import pytest

from fake_cudart import FakeLib
from test_paged import cache
from test_rotary import E4M3, append, attend, scales

from multi_lora_b200 import _native


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return FakeLib(tmp_path_factory.mktemp("fake"))


# of a cache of 8 blocks and 2 heads
@pytest.mark.parametrize("strides", [
    dict(k_head_stride=0), dict(v_head_stride=0), dict(k_block_stride=0), dict(v_block_stride=0), dict(k_block_stride=1),
    dict(v_block_stride=1, v_head_stride=7), dict(k_block_stride=0, k_head_stride=0),
])
def test_scales_that_share_memory_are_not_appended_to(strides):
    lib = _native.capi()
    assert append(lib, cache(dtype=E4M3), scales(**strides)) == -1
    assert b"share" in lib.mlora_last_error()


@pytest.mark.parametrize("c, strides", [
    ({}, {}), ({}, dict(k_block_stride=1, k_head_stride=8)), ({}, dict(v_block_stride=9, v_head_stride=3)),
    (dict(kv_heads=1), dict(k_head_stride=0, v_head_stride=0, k_block_stride=1)), (dict(num_blocks=1), dict(k_block_stride=0)),
    (dict(num_blocks=1, kv_heads=1), dict(k_block_stride=0, k_head_stride=0, v_block_stride=0, v_head_stride=0)),
])
def test_scales_apart_in_any_order_are(fake, c, strides):
    fake.reset()
    assert append(fake.c, cache(dtype=E4M3, k=4096, v=4096, **c), scales(**strides)) == 0, fake.error()


def test_attention_reads_scales_that_blocks_or_heads_share(fake):
    for strides in (dict(k_head_stride=0, v_head_stride=0), dict(k_block_stride=0, v_block_stride=0, k_head_stride=0)):
        fake.reset()
        assert attend(fake.c, cache(dtype=E4M3, k=4096, v=4096), scales(k=4096, v=4096, **strides)) == 0, fake.error()
