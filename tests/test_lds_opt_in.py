"""The opt-in of kernels with more than 64 KB of dynamic LDS (csrc/eg_lds.h) against stand-ins for the two HIP calls: once
for a kernel on a device, for every device, and again after a failure.  No kernel's attribute is set anywhere else."""
from __future__ import annotations

import subprocess

from tests.conftest import ROOT

CSRC = ROOT / "engraft-ngram_amd" / "csrc"

PROGRAM = r"""
#include "eg_lds.h"
#include <stdio.h>
static int device, calls;
static hipError_t answer = hipSuccess;
extern "C" hipError_t hipGetDevice(int* d) { *d = device; return hipSuccess; }
extern "C" hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { ++calls; return answer; }
#define EXPECT(x) if (!(x)) return fprintf(stderr, "line %d: " #x "\n", __LINE__), 1
int main() {
  const char kernels[2] = {};
  EXPECT(eg::allow_lds(kernels, 1) == hipSuccess && calls == 1);
  EXPECT(eg::allow_lds(kernels, 1) == hipSuccess && calls == 1);
  EXPECT(eg::allow_lds(kernels + 1, 1) == hipSuccess && calls == 2);
  device = 1;
  answer = hipErrorInvalidValue;
  EXPECT(eg::allow_lds(kernels, 1) == hipErrorInvalidValue && calls == 3);
  answer = hipSuccess;
  EXPECT(eg::allow_lds(kernels, 1) == hipSuccess && calls == 4);
  EXPECT(eg::allow_lds(kernels, 1) == hipSuccess && calls == 4);
  device = 0;
  EXPECT(eg::allow_lds(kernels, 1) == hipSuccess && calls == 4);
  return 0;
}
"""


def test_once_a_device_and_kernel(tmp_path):
    source, program = tmp_path / "opt_in.cpp", tmp_path / "opt_in"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-w", "-I", str(CSRC), "-I", "/opt/rocm/include", str(source),
                    "-o", str(program)], check=True, timeout=120)
    done = subprocess.run([str(program)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stderr


def test_no_attribute_is_set_elsewhere():
    using = [p.name for p in sorted(CSRC.iterdir()) if p.suffix in (".hip", ".h", ".cpp") and "hipFuncSetAttribute(" in p.read_text()]
    assert using == ["eg_lds.h"]
