// norm_grad.h -- descriptor and launchers of the residual LayerNorm operators
// (gsvdec_norm_*; kernels in norm_grad.cu).
//
// Per frame, over C channels:  s = x + y,  xh = (s - mean) rstd,
//   out = xh gamma + beta
//   a = dout gamma;  dx = rstd (a - mean(a) - xh mean(a xh))   (= dy)
//   dgamma = sum over frames of dout xh;  dbeta = sum of dout
// Frames t >= len[b] give out = 0, mean = rstd = 0, dx = 0 and add nothing.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "attn.h"

namespace gsv {

struct NormTensor {
  const void* p;
  int64_t b, o;  // element strides of the batch and of the outer axis (time, or channels)
};

struct NormArgs {
  Ty ty;
  bool rows;  // [B][T][C], channels contiguous; else [B][C][T], time contiguous
  int B, C, T;
  float eps;
  NormTensor x, y, out, dout, dx;
  const float *gamma, *beta;
  float *mean, *rstd;  // [B][T]
  const int* len;
  float *dgamma, *dbeta;
  float* part;  // backward workspace
  size_t ws_bytes;
};

constexpr int kNormRowsMaxC = 8192;
constexpr int kNormTimeMaxC = 2048;

size_t norm_bwd_workspace(const NormArgs& a);
cudaError_t norm_forward(const NormArgs& a, cudaStream_t st);
cudaError_t norm_backward(const NormArgs& a, cudaStream_t st);
// As attn_fwd_give_ups (attn.h).
cudaError_t norm_give_ups(int* out, cudaStream_t st);

}  // namespace gsv
