"""The LoRA apply paths on several devices of one process, on the library's host side with a runtime that has no GPU
(tests/fake_cudart.cpp): what a kernel is granted, it is granted on one device."""

from __future__ import annotations

import ctypes

import pytest

from fake_cudart import FakeLib

from multi_lora_b200 import _native


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return FakeLib(tmp_path_factory.mktemp("fake"))


def apply(fake, *, rank, rows, in_dim=4096, out_dim=4096, slots=8, segments=4):
    m = _native.MetadataT()
    m.bs, m.max_len, m.num_slots, m.scalings_dtype = segments, rows // segments, slots, 2
    m.seg_lens = m.seg_indptr = m.weight_indices = m.lora_ranks = m.scalings = 4096
    pointers = (ctypes.c_void_p * 1)(4096)
    dims, strides = (ctypes.c_int64 * 1)(out_dim), (ctypes.c_int64 * 1)(out_dim)
    return fake.c.mlora_apply_lora_group(4096, rows, in_dim, in_dim, 1, pointers, pointers, dims, pointers, strides, rank,
                                         ctypes.byref(m), 8192, rank, 0, None, None)


@pytest.mark.parametrize("path, number, rank, rows", [("fused", 1, 16, 64), ("fused", 1, 64, 8), ("stream", 3, 16, 256),
                                                      ("stream", 3, 64, 512), ("tc", 4, 64, 1024), ("tc", 4, 16, 512)])
def test_every_device_of_a_process(fake, path, number, rank, rows):
    fake.c.mlora_set_apply_path(_native.APPLY_PATHS[path])
    for dev in (2, 0, 5, 2):
        fake.reset()
        fake.device(dev)
        assert apply(fake, rank=rank, rows=rows) == 0, (dev, fake.error())
        assert fake.c.mlora_last_apply_path() == number
        assert {x.device for x in fake.launches()} == {dev} and all(x.result == 0 for x in fake.launches())


def test_a_device_that_refused_once_is_asked_again(fake):
    fake.c.mlora_set_apply_path(_native.APPLY_PATHS["fused"])
    fake.reset()
    fake.device(6)
    fake.c.fake_fail(8)  # every size of cluster: another path takes the call
    assert apply(fake, rank=16, rows=64) == 0 and fake.c.mlora_last_apply_path() != 1
    fake.c.fake_fail(0)
    assert apply(fake, rank=16, rows=64) == 0 and fake.c.mlora_last_apply_path() == 1
