// attn_common.cuh -- element access and row geometry shared by the attention kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>
#include <cstring>
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

// The first query with an allowed key (ql: none has); those before it may hold
// anything, so the backward reads them as zeros, like rows past ql.
__device__ __forceinline__ int first_query(int ql, int kl, int causal) {
  return kl == 0 ? ql : causal ? max(0, ql - kl) : 0;
}

// Eight channels as they lie in memory, turned into fp32 where they are used.
template <typename T>
struct Raw8 {
  uint4 u[sizeof(T) / 2];
  // Channels d0 .. d0 + 7 of a row, zeros from D on.
  __device__ __forceinline__ void load(const T* row, int d0, int D, bool vec) {
    if (vec) {
      const T* p = row + min(d0, D - 8);
#pragma unroll
      for (int k = 0; k < (int)sizeof(T) / 2; ++k) {
        u[k] = reinterpret_cast<const uint4*>(p)[k];
        if (d0 >= D) u[k] = make_uint4(0u, 0u, 0u, 0u);
      }
    } else {
      T e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = d0 + i < D ? row[d0 + i] : from_f<T>(0.f);
      memcpy(u, e, sizeof e);
    }
  }
  __device__ __forceinline__ void get(float* f) const {
    T e[8];
    memcpy(e, u, sizeof e);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f(e[i]);
  }
};

}  // namespace
}  // namespace gsv
