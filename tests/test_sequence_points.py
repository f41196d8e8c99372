"""fgm_api.hip holds no expression that reads and changes a value without an
order between the two (undefined, and silent under hipcc: attend_tree's cut of
its partial sums once divided by what the same expression incremented).  GCC
names them; the file is plain C++ but for the launch geometry, declared here."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "fastgemma_amd", "csrc")
ROCM = "/opt/rocm/include"

STUB = """#include <hip/hip_runtime.h>
extern const dim3 blockIdx, blockDim, threadIdx, gridDim;
"""


def problems(path: str, tmp_path) -> str:
    stub = tmp_path / "stub.h"
    stub.write_text(STUB)
    r = subprocess.run(["g++", "-std=c++17", "-x", "c++", "-fsyntax-only", "-Werror=sequence-point", "-D__HIP_PLATFORM_AMD__",
                        f"-I{ROCM}", "-include", str(stub), path], capture_output=True, text=True, timeout=300)
    return "" if r.returncode == 0 else r.stderr


pytestmark = pytest.mark.skipif(shutil.which("g++") is None or not os.path.isdir(ROCM), reason="no g++ or HIP headers")


def test_the_compiler_names_them(tmp_path):
    bad = tmp_path / "bad.hip"
    bad.write_text("struct S { int a, b; };\nvoid f(S& s) { s.a = (s.a + ++s.b - 1) / s.b; }\n")
    assert "sequence-point" in problems(str(bad), tmp_path)


def test_host_source(tmp_path):
    assert problems(os.path.join(CSRC, "fgm_api.hip"), tmp_path) == ""
