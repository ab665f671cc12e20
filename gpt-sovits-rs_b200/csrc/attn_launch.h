// attn_launch.h -- the attention kernels' launchers and the backward's workspace.
#pragma once
#include "attn.h"

namespace gsv {

// Query rows of one head whose relative gradients are one partial sum: the
// query tile of the tensor-core kernel, or a block of the fp32 one.
constexpr int kRelRows = 64, kRelRowsTensor = 128;
inline int64_t rel_blocks(const AttnArgs& a) {
  return (int64_t)a.B * a.H * cdiv(a.Tq, a.ty == Ty::F32 ? kRelRows : kRelRowsTensor);
}
constexpr float kHalfShift = 15.f;  // fp16 probabilities are carried as 2^15 p

// Backward workspace, all fp32: per query row (b, h, i) ndelta = -do . o and
// nlse2 = -lse log2(e), plus kHalfShift for fp16 (-inf for a row without keys,
// so that every exp2 of it is 0); for fp16 the norms |do_i| and |v_j| + max
// |relv|; per row and offset the products q . relk_r, do . relv_r (read by the
// score tiles); fp32: the near values of p and ds (written by the dq tiles);
// partial sums of the relative gradients.
struct BwdWs {
  float *ndelta, *nlse2, *ndo, *nv, *qrel, *grel, *pband, *sband, *part;
  size_t bytes;
};

inline BwdWs carve_bwd(const AttnArgs& a) {
  BwdWs w{};
  size_t at = 0;
  auto take = [&](size_t n) {
    float* p = reinterpret_cast<float*>(a.ws + at);
    at += (n * sizeof(float) + 255) / 256 * 256;
    return p;
  };
  const size_t rows = (size_t)a.B * a.H * a.Tq;
  w.ndelta = take(rows);
  w.nlse2 = take(rows);
  if (a.ty == Ty::F16) {
    w.ndo = take(rows);
    w.nv = take((size_t)a.B * a.Hkv * a.Tk);
  }
  if (a.nrel) {
    w.qrel = take(rows * a.nrel);
    w.grel = take(rows * a.nrel);
    if (a.ty == Ty::F32) {
      w.pband = take(rows * a.nrel);
      w.sband = take(rows * a.nrel);
    }
    w.part = take((size_t)rel_blocks(a) * 2 * a.nrel * a.D);
  }
  w.bytes = at;
  return w;
}

cudaError_t attn_fwd_tensor(const AttnArgs& a, cudaStream_t st);
cudaError_t attn_fwd_cores(const AttnArgs& a, cudaStream_t st);
cudaError_t attn_bwd_tensor(const AttnArgs& a, const BwdWs& ws, cudaStream_t st);
cudaError_t attn_bwd_cores(const AttnArgs& a, const BwdWs& ws, cudaStream_t st);
// ndelta, nlse2, the norms and the relative products of every row.
cudaError_t attn_bwd_rows(const AttnArgs& a, const BwdWs& ws, cudaStream_t st);
// drelk, drelv from the near values (fp32) or the query tiles' partial sums.
cudaError_t attn_bwd_rel(const AttnArgs& a, const BwdWs& ws, cudaStream_t st);

}  // namespace gsv
