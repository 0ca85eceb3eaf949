"""The library's objects linked against tests/fake_cudart.cpp: the C ABI on a host without a GPU, on any number of
devices that are not there."""

from __future__ import annotations

import ctypes
import subprocess
from dataclasses import dataclass
from typing import List

from multi_lora_b200 import _native, build


@dataclass
class Launch:
    device: int
    grid: tuple
    smem: int
    result: int


class FakeLib:
    def __init__(self, folder):
        objects = [build.OBJ / (src.stem + ".o") for src in sorted(build.CSRC.glob("*.cu"))]
        build.build_cuda_lib(force=not all(o.exists() for o in objects))
        path = folder / "libmlora_fake.so"
        subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-Wl,-Bsymbolic", "-I/usr/local/cuda/include",
                        str(build.ROOT / "tests" / "fake_cudart.cpp"), *map(str, objects), "-o", str(path)], check=True)
        self.c = ctypes.CDLL(str(path), mode=ctypes.RTLD_LOCAL)
        for name, (result, args) in _native.CAPI_SIGNATURES.items():
            f = getattr(self.c, name)
            f.restype, f.argtypes = result, args
        self.reset()

    def reset(self, sms: int = 148) -> None:
        self.c.fake_reset(sms)

    def device(self, index: int) -> None:
        self.c.fake_device(index)

    def launches(self) -> List[Launch]:
        out, row = [], (ctypes.c_int * 6)()
        for i in range(self.c.fake_launches()):
            self.c.fake_launch(i, row)
            out.append(Launch(row[0], tuple(row[1:4]), row[4], row[5]))
        return out

    def error(self) -> bytes:
        return self.c.mlora_last_error()
