"""What an append or a rotation writes has a place of its own: refusals of scales and rows that share memory (no GPU needed)."""

from __future__ import annotations

import pytest

from fake_cudart import FakeLib
from test_paged import cache
from test_rotary import E4M3, append, attend, rot, rotate, scales

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


# of 3 tokens of 2 (rotate) and 4 (append) heads of 64
@pytest.mark.parametrize("strides", [dict(ot=64, oh=64), dict(ot=64, oh=128), dict(ot=100, oh=64), dict(ot=0, oh=64), dict(ot=128, oh=0)])
def test_rotated_rows_that_overlap_are_refused(strides):
    lib = _native.capi()
    assert rotate(lib, **strides) == -1 and b"stride" in lib.mlora_last_error()
    assert append(lib, **strides) == -1 and b"stride" in lib.mlora_last_error()


@pytest.mark.parametrize("strides", [dict(ot=256, oh=64), dict(ot=64, oh=192), dict(ot=1000, oh=100), dict(ot=64, oh=1000)])
def test_rotated_rows_apart_in_any_order_are_not(fake, strides):
    fake.reset()
    assert rotate(fake.c, x=4096, **strides) == 0, fake.error()
    assert append(fake.c, cache(k=4096, v=4096), q=4096, **strides) == 0, fake.error()


def test_one_token_or_head_has_any_stride(fake):
    fake.reset()
    assert rotate(fake.c, rot(), tokens=1, ot=0) == 0 and rotate(fake.c, rot(), heads=1, oh=0, ot=64) == 0, fake.error()
