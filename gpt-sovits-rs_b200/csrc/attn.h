// attn.h -- descriptor and launchers of the attention operators
// (gsvdec_attention_*; kernels in attn_*.cu).
//
// For utterance b with ql valid queries and kl valid keys (clamped to Tq / Tk)
// the sequences are aligned at their ends: query i stands at key position
// pos = i + kl - ql.  Key j is allowed for it when j < kl and, with causal,
// j <= pos; both limits are one bound on j per row.  Offset r = j - pos is
// "near" when |r| <= window.
//   s_ij = scale q_i . (k_j + [near] relk_r)      p = softmax_j(s)
//   o_i  = sum_j p_ij (v_j + [near] relv_r)       lse_i = log sum_j exp(s_ij)
//   dp_ij = do_i . (v_j + [near] relv_r)          ds_ij = p_ij (dp_ij - do_i . o_i)
//   dq_i = scale sum_j ds_ij (k_j + [near] relk_r)
//   dk_j = scale sum_i ds_ij q_i                  dv_j = sum_i p_ij do_i
//   drelk_r = scale sum ds_{i, pos + r} q_i       drelv_r = sum p_{i, pos + r} do_i
// Rows with no allowed key, and rows i >= ql, give o = 0, lse = -inf, dq = 0.
// Key rows j >= kl are never read into a product and get dk = dv = 0.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "gsv_internal.h"

namespace gsv {

int ops_wait_selftest(int device, unsigned long long limit_ns, cudaStream_t st);  // ops_api.cu

enum class Ty { F32 = 0, F16 = 1, BF16 = 2 };  // GSV_DTYPE_*

constexpr int kAttnMaxD = 128;
constexpr int kAttnMaxWindow = 15;  // 2 * 15 + 1 offsets fit 32 rows of a tile

struct Str3 {
  int64_t b, h, t;  // element strides of batch, head, time; channels are contiguous
};

struct AttnArgs {
  Ty ty;
  int B, H, Hkv, Tq, Tk, D;
  int window, nrel;  // -1 and 0 without relative terms
  int causal;
  float scale;
  const void *q, *k, *v, *relk, *relv, *dout;
  const int *qlen, *klen;
  void *o, *dq, *dk, *dv, *drelk, *drelv;
  float* lse;  // [B][H][Tq]
  Str3 sq, sk, sv, so, sdo, sdq, sdk, sdv;
  char* ws;
  size_t ws_bytes;
  int* err;  // a handle's error word, for its give-ups; null: the operators' own counts
};

// Every row of the tensor starts on a 16-byte boundary and holds whole
// 16-byte vectors, so tiles can be moved by vectors.
inline bool attn_rows_aligned(const void* p, const Str3& s, int D, int elem) {
  const int64_t v = 16 / elem;
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s.b % v == 0 && s.h % v == 0 && s.t % v == 0 && D % v == 0;
}

// Workspace the call needs (0: none).
size_t attn_fwd_workspace(const AttnArgs& a);
size_t attn_bwd_workspace(const AttnArgs& a);
cudaError_t attn_forward(const AttnArgs& a, cudaStream_t st);
cudaError_t attn_backward(const AttnArgs& a, cudaStream_t st);
// Waits for the stream; *out: a count that has grown by at least one for every
// call without a handle in which a bounded device wait of the forward's
// (backward's) kernels on the current device gave up.
cudaError_t attn_fwd_give_ups(int* out, cudaStream_t st);
cudaError_t attn_bwd_give_ups(int* out, cudaStream_t st);
// One bounded wait that nothing completes, reported as the forward's kernels
// report theirs (gsvdec_selftest_attention_wait).
cudaError_t attn_wait_selftest(const AttnArgs& a, unsigned long long limit_ns, cudaStream_t st);

}  // namespace gsv
