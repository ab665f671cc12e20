// kernel_setup.h -- launch setup of a kernel, done once per (kernel, device)
// instead of per launch: the shared-memory carveout, the register count, and
// the dynamic shared-memory limit (raised only when a launch needs more).
// Short launches (the flow's) were bound by these host calls.
//
// The limit is process-wide state of the kernel, and a launch follows its
// setup outside the lock: it must never be lowered, or another host thread's
// launch of the same kernel may find it below its own size.
#pragma once
#include <cuda_runtime.h>

#include <mutex>

namespace gsv {
namespace {

// Slots per device and kernel signature: every instantiation of a kernel
// template shares one signature (the norm's row kernel has 72, the tap GEMM a
// few dozen).  Kernels past the slots are set up at every launch.
constexpr int kSetupSlots = 128;

template <typename K>
cudaError_t kernel_setup(K kern, size_t smem, int* regs) {
  struct Entry {
    int regs = 0, smem = 0;
    bool ready = false;
  };
  static std::mutex mu;
  static Entry table[64][kSetupSlots];
  static const void* keys[64][kSetupSlots] = {};
  const void* fn = (const void*)kern;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  std::lock_guard<std::mutex> lock(mu);
  Entry* en = nullptr;
  for (int i = 0; i < kSetupSlots && !en; ++i) {
    if (keys[dev][i] == fn) en = &table[dev][i];
    else if (!keys[dev][i]) {
      keys[dev][i] = fn;
      en = &table[dev][i];
    }
  }
  Entry scratch;
  const bool kept = en != nullptr;
  if (!kept) en = &scratch;
  if (!en->ready) {
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout,
                                         cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return e;
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, fn);
    if (e != cudaSuccess) return e;
    en->regs = fa.numRegs;
    if (!kept) en->smem = fa.maxDynamicSharedSizeBytes;  // what an earlier launch set
    en->ready = true;
  }
  if ((int)smem > en->smem) {
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    en->smem = (int)smem;
  }
  *regs = en->regs;
  return cudaSuccess;
}

}  // namespace
}  // namespace gsv
