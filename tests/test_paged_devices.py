"""The launches of the paged step on the library's host side, with a runtime that has no GPU (tests/fake_cudart.cpp):
grids that are not empty, and what each kernel needs on each device of a process."""

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


def plan(fake, requests):
    return fake.c.mlora_plan_paged_step(16, 16, 16, requests, 16, 4, 16, 16, 4, 4, 16, 16, 16, 16, 16, 16, 16, 8, 16, None,
                                        None)


@pytest.mark.parametrize("call", [
    lambda f: attend(f), lambda f: attend(f, width=4000), lambda f: attend(f, rows=300, most=90),
    lambda f: attend(f, rows=300, most=90, dim=128, dtype=1), lambda f: attend(f, dtype=2), lambda f: plan(f, 8192),
], ids=["cluster", "dealt", "chunk", "chunk-f16-128", "general", "plan"])
def test_every_device_of_a_process(fake, call):
    """Shared memory above the 48 KB that a launch has by itself is granted for a kernel on one device."""
    for dev in (3, 1, 0, 3, 2, 1):
        fake.reset()
        fake.device(dev)
        assert call(fake) == 0, (dev, fake.error())
        assert [x.device for x in fake.launches()] == [dev]
        fake.reset()
        fake.device(dev)
        assert call(fake) == 0 and fake.c.fake_attribute_calls() == 0  # granted by now: nothing is asked again


def test_a_device_that_refused_once_is_asked_again(fake):
    fake.reset()
    fake.device(7)
    fake.c.fake_fail(2)
    assert attend(fake, width=4000) != 0 and attend(fake, width=4000) != 0 and not fake.launches()
    assert attend(fake, width=4000) == 0 and fake.launches()[0].result == 0


def test_a_grid_has_the_device_s_own_sms(fake):
    fake.reset()
    for dev, sms in ((8, 148), (9, 132), (8, 148), (9, 132)):
        fake.c.fake_sms(dev, sms)
        fake.device(dev)
        assert attend(fake, width=4000) == 0 and attend(fake, rows=300, most=90) == 0
        assert [x.grid[0] for x in fake.launches()[-2:]] == [2 * sms, sms]
