"""kernel_setup (csrc/kernel_setup.h) against a stand-in for the CUDA runtime:
a kernel's shared-memory limit is never lowered, however many kernels share a
signature, and a kernel that is set up already costs no further calls."""
from __future__ import annotations

import subprocess

import pytest

from conftest import ROOT

HARNESS = r"""
#include "kernel_setup.h"

#include <cstdio>
#include <map>
#include <string>

static std::map<const void*, int> limits;
static int calls = 0, lowered = 0;

extern "C" {
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaFuncGetAttributes(cudaFuncAttributes* a, const void* f) {
  ++calls;
  *a = cudaFuncAttributes{};
  a->numRegs = 32;
  a->maxDynamicSharedSizeBytes = limits.count(f) ? limits[f] : 48 * 1024;
  return cudaSuccess;
}
cudaError_t cudaFuncSetAttribute(const void* f, cudaFuncAttribute which, int v) {
  ++calls;
  if (which == cudaFuncAttributeMaxDynamicSharedMemorySize) {
    if (limits.count(f) && v < limits[f]) ++lowered;
    limits[f] = v;
  }
  return cudaSuccess;
}
}

using Kernel = void (*)(int);
static char place[300];  // as many kernels of one signature, told apart by their addresses

int main(int, char** argv) {
  const int kernels = std::stoi(argv[1]);
  int short_of = 0;
  for (const int smem : {100000, 20000, 60000, 120000, 0}) {
    for (int k = 0; k < kernels; ++k) {
      const Kernel f = reinterpret_cast<Kernel>(place + k);
      int regs = 0;
      if (gsv::kernel_setup(f, smem, &regs) != cudaSuccess || regs != 32) return 1;
      if (limits[(const void*)f] < smem) ++short_of;
    }
  }
  int regs = 0;
  const int again = calls;
  gsv::kernel_setup(reinterpret_cast<Kernel>(place), 100000, &regs);
  std::printf("%d %d %d\n", short_of, lowered, calls - again);
  return 0;
}
"""


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    d = tmp_path_factory.mktemp("setup")
    (d / "h.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-I", str(ROOT / "gpt-sovits-rs_b200" / "csrc"), "-I",
                    "/usr/local/cuda/include", str(d / "h.cpp"), "-o", str(d / "h"), "-lpthread"], check=True)
    return d / "h"


@pytest.mark.parametrize("kernels", [1, 72, 300])
def test_the_limit_is_never_lowered(harness, kernels):
    out = subprocess.run([str(harness), str(kernels)], check=True, capture_output=True, text=True).stdout
    short_of, lowered, again = map(int, out.split())
    assert short_of == 0 and lowered == 0
    assert again == 0  # one that has a slot
