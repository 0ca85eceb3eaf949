"""The launches of the paged step on the library's host side, with a runtime that has no GPU (tests/fake_cudart.cpp):
grids that are not empty."""

from __future__ import annotations

import ctypes

import pytest

from fake_cudart import FakeLib
from test_paged import cache

from multi_lora_b200 import paged_kv


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return FakeLib(tmp_path_factory.mktemp("fake"))


def attend(fake, *, requests=3, rows=12, width=4, most=1, dim=64, dtype=0, heads=4):
    c = cache(head_dim=dim, dtype=dtype, k=4096, v=4096)
    for side in "kv":
        for name, value in (("block", 16 * 2 * dim), ("slot", 2 * dim), ("head", dim)):
            setattr(c, f"{side}_{name}_stride", value)
    return fake.c.mlora_paged_attention(4096, heads * dim, dim, rows, heads, ctypes.byref(c), 4096, width, width, 4096,
                                        4096, requests, most, 1.0, 0, 4096, heads * dim, dim, 4096,
                                        paged_kv.ATTENTION_WORKSPACE_BYTES, None, None)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("width", [0, 4, 256, 4000])
@pytest.mark.parametrize("requests, rows, most", [(0, 5, 1), (0, 5, 0), (0, 300, 100), (1, 5, 1), (40, 50, 1), (40, 300, 90)])
def test_every_attention_launch_has_blocks(fake, requests, rows, most, width, dtype):
    fake.reset()
    assert attend(fake, requests=requests, rows=rows, most=most, width=width, dtype=dtype) == 0, fake.error()
    launches = fake.launches()
    assert len(launches) == 1 and launches[0].result == 0 and min(launches[0].grid) > 0
