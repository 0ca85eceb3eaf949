"""The operators' library in a C++ process: it needs torch's C++ libraries and no Python (no GPU needed)."""

from __future__ import annotations

import os
import subprocess
from pathlib import Path

import torch

from multi_lora_b200 import _native

PROGRAM = r"""
#include <dlfcn.h>
#include <stdio.h>
int main(int, char** argv) {
  if (dlopen(argv[1], RTLD_NOW | RTLD_GLOBAL) == nullptr) {
    fprintf(stderr, "%s\n", dlerror());
    return 1;
  }
  return dlsym(RTLD_DEFAULT, "Py_IsInitialized") != nullptr ? 2 : 0;  // an interpreter came along
}
"""


def test_a_process_without_python_loads_the_operators(tmp_path):
    source, program = tmp_path / "load.cpp", tmp_path / "load"
    source.write_text(PROGRAM)
    subprocess.run(["g++", str(source), "-o", str(program), "-ldl"], check=True)
    env = dict(os.environ, LD_LIBRARY_PATH=str(Path(torch.__file__).parent / "lib"))
    run = subprocess.run([str(program), str(_native.TORCH_LIB_PATH)], env=env, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
