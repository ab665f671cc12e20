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

// Backward workspace, all fp32.  Query rows of a head are grouped in blocks of
// kRowBlock, the last one filled up (their number even), so that a block's
// values are one aligned run that a bulk copy can move:
//   rows  [b][h][block][2][kRowBlock]: nlse2 = -lse log2(e), plus kHalfShift
//         for fp16, and ndelta = -do . o; -inf and 0 for a row without keys or
//         past Tq, so that every exp2 of it is 0
//   rel   [b][h][block][2][kRowBlock][nrel]: q . relk_r and do . relv_r
// fp16: the norms |do_i| [b][h][Tq] and |v_j| + max |relv| [b][hk][Tk].  fp32
// with a window: the near values of p and ds [b][h][Tq][nrel], written by the
// dq tiles.  part: partial sums of the relative gradients.
constexpr int kRowBlock = 64;
struct BwdWs {
  float *rows, *rel, *ndo, *nv, *pband, *sband, *part;
  int blocks;  // row blocks of a head
  size_t bytes;
};

// nlse2 of row i of head bh (ndelta kRowBlock later), and its run of q . relk_r
// (do . relv_r kRowBlock nrel later).
__host__ __device__ inline float* row_at(const BwdWs& w, int64_t bh, int i) {
  return w.rows + ((bh * w.blocks + i / kRowBlock) * 2) * kRowBlock + i % kRowBlock;
}
__host__ __device__ inline float* rel_at(const BwdWs& w, int64_t bh, int i, int nrel) {
  return w.rel + (((bh * w.blocks + i / kRowBlock) * 2) * kRowBlock + i % kRowBlock) * nrel;
}

inline BwdWs carve_bwd(const AttnArgs& a) {
  BwdWs w{};
  size_t at = 0;
  auto take = [&](size_t n) {
    float* p = reinterpret_cast<float*>(a.ws + at);
    at += (n * sizeof(float) + 255) / 256 * 256;
    return p;
  };
  const size_t rows = (size_t)a.B * a.H * a.Tq;
  w.blocks = cdiv(a.Tq, 2 * kRowBlock) * 2;
  const size_t padded = (size_t)a.B * a.H * w.blocks * kRowBlock;
  w.rows = take(2 * padded);
  if (a.ty == Ty::F16) {
    w.ndo = take(rows);
    w.nv = take((size_t)a.B * a.Hkv * a.Tk);
  }
  if (a.nrel) {
    w.rel = take(2 * padded * a.nrel);
    if (a.ty == Ty::F32) {
      w.pband = take(rows * a.nrel);
      w.sband = take(rows * a.nrel);
    }
    w.part = take((size_t)rel_blocks(a) * 2 * a.nrel * a.D);
  }
  w.bytes = at;
  return w;
}

// The row pass: G lanes share a row, and a block of kRowThreads takes kRowTurns
// rows per group.  Query rows of all heads come first, then (fp16, for the
// norms of v) the key rows of all key heads.
constexpr int kRowThreads = 256, kRowTurns = 2;
inline int row_lanes(int D) { return D <= 32 ? 4 : D <= 64 ? 8 : 16; }
struct RowBlocks {
  int64_t q, k;
};
inline RowBlocks row_blocks(const AttnArgs& a) {
  const int rows = kRowThreads / row_lanes(a.D) * kRowTurns, padded = cdiv(a.Tq, 2 * kRowBlock) * 2 * kRowBlock;
  return {(int64_t)cdiv(padded, rows) * a.H * a.B, a.ty == Ty::F16 ? (int64_t)cdiv(a.Tk, rows) * a.Hkv * a.B : 0};
}

// Most blocks of a launch of the call.  Tiles are split over several blocks
// only where there are few of them, so they do not add to it.
inline int64_t attn_most_blocks(const AttnArgs& a, bool bwd) {
  const int tile = a.ty == Ty::F32 ? 64 : 128;
  const int64_t q = (int64_t)cdiv(a.Tq, tile) * a.H * a.B;
  if (!bwd) return q;
  const RowBlocks r = row_blocks(a);
  const int64_t main = q + (int64_t)cdiv(a.Tk, tile) * a.Hkv * a.B;
  return main > r.q + r.k ? main : r.q + r.k;
}

constexpr int kFewRows = 8;  // most rows per key head of attn_fwd_few_rows
cudaError_t attn_fwd_few_rows(const AttnArgs& a, cudaStream_t st);
cudaError_t attn_fwd_tensor(const AttnArgs& a, cudaStream_t st);
cudaError_t attn_fwd_cores(const AttnArgs& a, cudaStream_t st);
cudaError_t attn_bwd_tensor(const AttnArgs& a, const BwdWs& ws, cudaStream_t st);
cudaError_t attn_bwd_cores(const AttnArgs& a, const BwdWs& ws, cudaStream_t st);
// The rows, rel, ndo and nv parts of the workspace.
cudaError_t attn_bwd_rows(const AttnArgs& a, const BwdWs& ws, cudaStream_t st);
// drelk, drelv from the near values (fp32) or the query tiles' partial sums.
cudaError_t attn_bwd_rel(const AttnArgs& a, const BwdWs& ws, cudaStream_t st);

}  // namespace gsv
