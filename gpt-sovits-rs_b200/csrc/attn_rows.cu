// attn_rows.cu -- the attention backward's per-row pass and the gradients of
// the relative keys and values, and the choice of kernels of both directions.
#include <algorithm>

#include "attn_common.cuh"
#include "attn_launch.h"

namespace gsv {
namespace {

constexpr int kRowWarps = 8;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// One warp per query row.  delta = do . o in fp32; lane r then holds offset r's
// products with the row, read from shared memory, against relk / relv rows of
// odd pitch (no bank conflicts between lanes).  fp16 (F16) adds the norms of
// the rows of do and v.
template <typename T>
__global__ void __launch_bounds__(kRowWarps * 32) bwd_rows_kernel(const AttnArgs a, const BwdWs ws) {
  extern __shared__ float sm[];
  const int D = a.D, L = D | 1, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  float* srk = sm;
  float* srv = srk + a.nrel * L;
  float* sq = srv + a.nrel * L + w * 2 * D;
  float* sg = sq + D;
  for (int e = threadIdx.x; e < a.nrel * D; e += blockDim.x) {
    const int r = e / D, d = e - r * D;
    srk[r * L + d] = to_f(static_cast<const T*>(a.relk)[e]);
    srv[r * L + d] = to_f(static_cast<const T*>(a.relv)[e]);
  }
  __syncthreads();
  constexpr bool F16 = std::is_same<T, __half>::value;
  const int64_t rows = (int64_t)a.B * a.H * a.Tq;
  if (F16) {
    float ev = 0.f;  // largest |relv|^2
    if (lane < a.nrel)
      for (int d = 0; d < D; ++d) ev = fmaf(srv[lane * L + d], srv[lane * L + d], ev);
    ev = sqrtf(warp_max(ev));
    const int64_t keys = (int64_t)a.B * a.Hkv * a.Tk;
    for (int64_t row = (int64_t)blockIdx.x * kRowWarps + w; row < keys; row += (int64_t)gridDim.x * kRowWarps) {
      const int j = (int)(row % a.Tk), h = (int)(row / a.Tk % a.Hkv), b = (int)(row / a.Tk / a.Hkv);
      if (j >= clamp_len(a.klen, b, a.Tk)) continue;
      const T* v = static_cast<const T*>(a.v) + b * a.sv.b + h * a.sv.h + j * a.sv.t;
      float s = 0.f;
      for (int d = lane; d < D; d += 32) s = fmaf(to_f(v[d]), to_f(v[d]), s);
      s = warp_sum(s);
      if (lane == 0) ws.nv[row] = sqrtf(s) + ev;
    }
  }
  for (int64_t row = (int64_t)blockIdx.x * kRowWarps + w; row < rows; row += (int64_t)gridDim.x * kRowWarps) {
    const int i = (int)(row % a.Tq), h = (int)(row / a.Tq % a.H), b = (int)(row / a.Tq / a.H);
    const int ql = clamp_len(a.qlen, b, a.Tq), kl = clamp_len(a.klen, b, a.Tk);
    if (allowed_keys(i, ql, kl, a.causal) == 0) {
      if (lane == 0) {
        ws.delta[row] = 0.f;
        ws.lse2[row] = INFINITY;
        if (F16) ws.ndo[row] = 0.f;
      }
      if (lane < a.nrel) ws.qrel[row * a.nrel + lane] = ws.grel[row * a.nrel + lane] = 0.f;
      continue;
    }
    const T* g = static_cast<const T*>(a.dout) + b * a.sdo.b + h * a.sdo.h + i * a.sdo.t;
    const T* o = static_cast<const T*>(a.o) + b * a.so.b + h * a.so.h + i * a.so.t;
    const T* q = static_cast<const T*>(a.q) + b * a.sq.b + h * a.sq.h + i * a.sq.t;
    float s = 0.f, gg = 0.f;
    for (int d = lane; d < D; d += 32) {
      const float gv = to_f(g[d]);
      s = fmaf(gv, to_f(o[d]), s);
      if (F16) gg = fmaf(gv, gv, gg);
      if (a.nrel) {
        sg[d] = gv;
        sq[d] = to_f(q[d]);
      }
    }
    s = warp_sum(s);
    if (F16) gg = warp_sum(gg);
    if (lane == 0) {
      ws.delta[row] = s;
      ws.lse2[row] = a.lse[row] * kLog2e;
      if (F16) ws.ndo[row] = sqrtf(gg);
    }
    __syncwarp();
    if (lane < a.nrel) {
      float x = 0.f, y = 0.f;
      for (int d = 0; d < D; ++d) {
        x = fmaf(sq[d], srk[lane * L + d], x);
        y = fmaf(sg[d], srv[lane * L + d], y);
      }
      ws.qrel[row * a.nrel + lane] = x;
      ws.grel[row * a.nrel + lane] = y;
    }
    __syncwarp();
  }
}

// Partial sums over a block's run of rows: thread d holds channel d of every
// offset (NR of them).  Fixed row order, so the result does not depend on
// scheduling.
template <typename T, int NR>
__global__ void __launch_bounds__(kAttnMaxD) bwd_rel_kernel(const AttnArgs a, const BwdWs ws, const int64_t per) {
  const int d = threadIdx.x, D = a.D;
  const int64_t rows = (int64_t)a.B * a.H * a.Tq;
  const int64_t r0 = blockIdx.x * per, r1 = min(rows, r0 + per);
  float ak[NR] = {}, av[NR] = {};
  for (int64_t row = r0; row < r1; ++row) {
    const int i = (int)(row % a.Tq), h = (int)(row / a.Tq % a.H), b = (int)(row / a.Tq / a.H);
    const int ql = clamp_len(a.qlen, b, a.Tq), kl = clamp_len(a.klen, b, a.Tk);
    const int n = allowed_keys(i, ql, kl, a.causal);
    if (n == 0) continue;
    const int base = i + kl - ql - a.window;  // key of offset 0
    float q = 0.f, g = 0.f;
    if (d < D) {
      q = to_f(static_cast<const T*>(a.q)[b * a.sq.b + h * a.sq.h + i * a.sq.t + d]);
      g = to_f(static_cast<const T*>(a.dout)[b * a.sdo.b + h * a.sdo.h + i * a.sdo.t + d]);
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      if (r >= a.nrel || base + r < 0 || base + r >= n) continue;
      ak[r] = fmaf(ws.sband[row * a.nrel + r], q, ak[r]);
      av[r] = fmaf(ws.pband[row * a.nrel + r], g, av[r]);
    }
  }
  if (d >= D) return;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    if (r >= a.nrel) continue;
    ws.part[((int64_t)blockIdx.x * 2 * a.nrel + r) * D + d] = ak[r] * a.scale;
    ws.part[((int64_t)blockIdx.x * 2 * a.nrel + a.nrel + r) * D + d] = av[r];
  }
}

template <typename T>
__global__ void bwd_rel_sum_kernel(const AttnArgs a, const BwdWs ws, const int blocks) {
  const int n = a.nrel * a.D, e = blockIdx.x * blockDim.x + threadIdx.x;
  if (e >= 2 * n) return;
  float s = 0.f;
  for (int x = 0; x < blocks; ++x) s += ws.part[(int64_t)x * 2 * n + e];
  if (e < n) static_cast<T*>(a.drelk)[e] = from_f<T>(s);
  else static_cast<T*>(a.drelv)[e - n] = from_f<T>(s);
}

template <typename T>
cudaError_t rows_t(const AttnArgs& a, const BwdWs& ws, cudaStream_t st) {
  const int64_t rows = (int64_t)a.B * a.H * a.Tq;
  const int grid = (int)std::min<int64_t>((rows + kRowWarps - 1) / kRowWarps, 148 * 8);
  const size_t smem = sizeof(float) * (2 * a.nrel * (a.D | 1) + kRowWarps * 2 * a.D);
  bwd_rows_kernel<T><<<grid, kRowWarps * 32, smem, st>>>(a, ws);
  return cudaGetLastError();
}

template <typename T>
cudaError_t rel_t(const AttnArgs& a, const BwdWs& ws, cudaStream_t st) {
  const int64_t rows = (int64_t)a.B * a.H * a.Tq;
  const int64_t per = std::max<int64_t>(1, (rows + kRelBlocks - 1) / kRelBlocks);
  const int blocks = (int)std::max<int64_t>(1, (rows + per - 1) / per);
  if (a.nrel <= 9) bwd_rel_kernel<T, 9><<<blocks, kAttnMaxD, 0, st>>>(a, ws, per);
  else bwd_rel_kernel<T, 2 * kAttnMaxWindow + 1><<<blocks, kAttnMaxD, 0, st>>>(a, ws, per);
  bwd_rel_sum_kernel<T><<<cdiv(2 * a.nrel * a.D, 128), 128, 0, st>>>(a, ws, blocks);
  return cudaGetLastError();
}

}  // namespace

cudaError_t attn_bwd_rows(const AttnArgs& a, const BwdWs& ws, cudaStream_t st) {
  if (a.ty == Ty::F32) return rows_t<float>(a, ws, st);
  return a.ty == Ty::F16 ? rows_t<__half>(a, ws, st) : rows_t<__nv_bfloat16>(a, ws, st);
}

cudaError_t attn_bwd_rel(const AttnArgs& a, const BwdWs& ws, cudaStream_t st) {
  if (a.ty == Ty::F32) return rel_t<float>(a, ws, st);
  return a.ty == Ty::F16 ? rel_t<__half>(a, ws, st) : rel_t<__nv_bfloat16>(a, ws, st);
}

size_t attn_fwd_workspace(const AttnArgs&) { return 0; }
size_t attn_bwd_workspace(const AttnArgs& a) { return carve_bwd(a).bytes; }

cudaError_t attn_forward(const AttnArgs& a, cudaStream_t st) {
  if (!a.Tq) return cudaSuccess;
  return a.ty == Ty::F32 ? attn_fwd_cores(a, st) : attn_fwd_tensor(a, st);
}

cudaError_t attn_backward(const AttnArgs& a, cudaStream_t st) {
  const BwdWs ws = carve_bwd(a);
  cudaError_t e = a.Tq ? attn_bwd_rows(a, ws, st) : cudaSuccess;
  if (e == cudaSuccess && (a.Tq || a.Tk)) e = a.ty == Ty::F32 ? attn_bwd_cores(a, ws, st) : attn_bwd_tensor(a, ws, st);
  if (e == cudaSuccess && a.nrel) e = attn_bwd_rel(a, ws, st);
  return e;
}

}  // namespace gsv
