"""CPU: settings of kernels are made on every device that launches them, not on the first one alone."""
import os
import re
import shutil
import subprocess

import pytest

from tests.conftest import PKG_NAME, ROOT

CSRC = os.path.join(ROOT, PKG_NAME, "csrc")

PROGRAM = r"""
#include "per_device.h"
#include <cstdio>
#include <cstring>
static int device, fail_on = -1;
static char calls[4096];
extern "C" cudaError_t cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void* f, cudaFuncAttribute a, int bytes) {
  if (device == fail_on) return cudaErrorInvalidValue;
  std::snprintf(calls + std::strlen(calls), 64, "%c%d:%d ", f == (const void*)&device ? 'a' : 'b', device, bytes);
  return a == cudaFuncAttributeMaxDynamicSharedMemorySize ? cudaSuccess : cudaErrorInvalidValue;
}
using namespace b200moe;
static cudaError_t first(int dev) {
  static PerDevice done;
  device = dev;
  return allow_smem(done, (const void*)&device, 100);
}
static cudaError_t second(int dev) {
  static PerDevice done;
  device = dev;
  return allow_smem(done, (const void*)&fail_on, 200);
}
int main() {
  int bad = 0;
  for (int dev : {0, 1, 0, 1, 63, 63}) bad += first(dev) != cudaSuccess;
  fail_on = 2;
  bad += second(2) != cudaErrorInvalidValue;
  fail_on = -1;
  for (int dev : {2, 2, 0, 64, 64}) bad += second(dev) != cudaSuccess;
  std::printf("%d %s", bad, calls);
}
"""


@pytest.mark.skipif(shutil.which("g++") is None or not os.path.exists("/usr/local/cuda/include/cuda_runtime.h"), reason="no compiler or no CUDA headers")
def test_once_on_each_device(tmp_path):
    src = tmp_path / "p.cpp"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-I", CSRC, "-I", "/usr/local/cuda/include", str(src), "-o", str(tmp_path / "p")], check=True)
    out = subprocess.run([str(tmp_path / "p")], check=True, capture_output=True, text=True).stdout
    assert out.split() == ["0", "a0:100", "a1:100", "a63:100", "b2:200", "b0:200", "b64:200", "b64:200"]


def test_no_kernel_is_set_up_another_way():
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".cu", ".cuh")):
            text = open(os.path.join(CSRC, name)).read()
            assert "cudaFuncSetAttribute" not in text, name
            assert len(re.findall(r"\ballow_smem\(", text)) == len(re.findall(r"static PerDevice \w+;", text)), name
