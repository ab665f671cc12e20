// attn_common.cuh -- element access and row geometry shared by the attention kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>
#include <type_traits>

#include "attn.h"

namespace gsv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Valid lengths of utterance b, clamped to the tensors.
__device__ __forceinline__ int clamp_len(const int* len, int b, int T) {
  return len ? min(max(len[b], 0), T) : T;
}

// Number of allowed keys of query i (they are the keys 0 .. n - 1).
__device__ __forceinline__ int allowed_keys(int i, int ql, int kl, int causal) {
  if (i >= ql) return 0;
  return causal ? min(kl, max(0, i + kl - ql + 1)) : kl;
}

}  // namespace
}  // namespace gsv
