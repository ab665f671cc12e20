// attn_simt.cu -- attention forward and backward on the CUDA cores, fp32
// arithmetic throughout (formulas in attn.h).
//
// One block of 256 threads works on 64 x 64 score tiles; a thread holds 4 x 4
// scores (rows 4 ty .., columns tx + 16 c) and 4 rows x D / 16 columns of each
// accumulator.  All operand tiles stay row-major in shared memory with a row
// pitch of D + 4 floats: a quarter warp reading float4s of consecutive rows
// then hits all 32 banks once.  Score products read 8 float4 for 64 FMAs,
// which keeps shared memory (12 wavefronts) below the FMA time (16 cycles).
// The forward walks the key tiles once with a running maximum and sum; the
// backward recomputes the probabilities from the saved log-sum-exp, once per
// key tile (dk, dv) and once per query tile (dq), so every gradient element
// is summed by one thread in a fixed order.
#include <algorithm>

#include "attn_common.cuh"
#include "attn_launch.h"

namespace gsv {
namespace {

constexpr int kBT = 64;        // rows and columns of a score tile
constexpr int kThreads = 256;
constexpr int kLdP = kBT + 4;  // pitch of a transposed probability tile

// rows x DP floats from global rows (nvalid of them, D channels), zeros elsewhere.
template <typename T, int DP>
__device__ __forceinline__ void load_rows(float* s, const T* g, int64_t stride, int nvalid, int D, bool vec) {
  constexpr int V = DP / 4;
  for (int i = threadIdx.x; i < kBT * V; i += kThreads) {
    const int r = i / V, c = (i - r * V) * 4;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < nvalid && c < D) {
      const T* p = g + (int64_t)r * stride + c;
      if (vec && sizeof(T) == 4) {
        o = *reinterpret_cast<const float4*>(p);
      } else {
        o.x = to_f(p[0]);
        if (c + 1 < D) o.y = to_f(p[1]);
        if (c + 2 < D) o.z = to_f(p[2]);
        if (c + 3 < D) o.w = to_f(p[3]);
      }
    }
    *reinterpret_cast<float4*>(s + r * (DP + 4) + c) = o;
  }
}

// acc[a][c] += A[4 ty + a] . B[tx + 16 c]
template <int DP>
__device__ __forceinline__ void dot_tile(const float* A, const float* B, int ty, int tx, float acc[4][4]) {
  constexpr int L = DP + 4;
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    float4 x[4], y[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) x[a] = *reinterpret_cast<const float4*>(A + (4 * ty + a) * L + d);
#pragma unroll
    for (int c = 0; c < 4; ++c) y[c] = *reinterpret_cast<const float4*>(B + (tx + 16 * c) * L + d);
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        acc[a][c] = fmaf(x[a].x, y[c].x, acc[a][c]);
        acc[a][c] = fmaf(x[a].y, y[c].y, acc[a][c]);
        acc[a][c] = fmaf(x[a].z, y[c].z, acc[a][c]);
        acc[a][c] = fmaf(x[a].w, y[c].w, acc[a][c]);
      }
  }
}

// acc[a][w] += sum_j P[j][4 ty + a] M[j][tx W + w], W = DP / 16
template <int DP>
__device__ __forceinline__ void acc_tile(const float* P, const float* M, int ty, int tx, float (*acc)[DP / 16]) {
  constexpr int L = DP + 4, W = DP / 16;
#pragma unroll 4
  for (int j = 0; j < kBT; ++j) {
    const float4 p = *reinterpret_cast<const float4*>(P + j * kLdP + 4 * ty);
    float m[W];
#pragma unroll
    for (int w = 0; w < W; w += 2) {
      const float2 t = *reinterpret_cast<const float2*>(M + j * L + tx * W + w);
      m[w] = t.x;
      m[w + 1] = t.y;
    }
#pragma unroll
    for (int w = 0; w < W; ++w) {
      acc[0][w] = fmaf(p.x, m[w], acc[0][w]);
      acc[1][w] = fmaf(p.y, m[w], acc[1][w]);
      acc[2][w] = fmaf(p.z, m[w], acc[2][w]);
      acc[3][w] = fmaf(p.w, m[w], acc[3][w]);
    }
  }
}

__device__ __forceinline__ float row_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int DP>
__host__ __device__ constexpr int tile_floats() { return kBT * (DP + 4); }

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) attn_fwd_simt(const AttnArgs a, const bool vec) {
  constexpr int W = DP / 16;
  extern __shared__ __align__(16) float sm[];
  float* sQ = sm;
  float* sK = sQ + tile_floats<DP>();
  float* sV = sK + tile_floats<DP>();
  float* sP = sV + tile_floats<DP>();
  float* sR = sP + kBT * kLdP;  // [nrel][64]: q . relk, then the near scores
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int i0 = blockIdx.x * kBT, h = blockIdx.y, b = blockIdx.z;
  const int ql = clamp_len(a.qlen, b, a.Tq), kl = clamp_len(a.klen, b, a.Tk), off = kl - ql;
  const int hk = h / (a.H / a.Hkv), D = a.D;
  const T* q = static_cast<const T*>(a.q) + b * a.sq.b + h * a.sq.h + (int64_t)i0 * a.sq.t;
  const T* k = static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h;
  const T* v = static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h;
  load_rows<T, DP>(sQ, q, a.sq.t, ql - i0, D, vec);
  __syncthreads();
  const T* relk = static_cast<const T*>(a.relk);
  const T* relv = static_cast<const T*>(a.relv);
  for (int e = threadIdx.x; e < a.nrel * kBT; e += kThreads) {
    const int r = e / kBT, i = e - r * kBT;
    float s = 0.f;
    for (int d = 0; d < D; ++d) s = fmaf(sQ[i * (DP + 4) + d], to_f(relk[(int64_t)r * D + d]), s);
    sR[e] = s;
  }
  float acc[4][W] = {}, m[4], l[4] = {};
  int n[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    m[x] = -INFINITY;
    n[x] = allowed_keys(i0 + 4 * ty + x, ql, kl, a.causal);
  }
  const int last = min(i0 + kBT, ql) - 1;
  const int kend = last < i0 ? 0 : allowed_keys(last, ql, kl, a.causal);
  const float sl2 = a.scale * kLog2e;
  for (int j0 = 0; j0 < kend; j0 += kBT) {
    __syncthreads();
    load_rows<T, DP>(sK, k + (int64_t)j0 * a.sk.t, a.sk.t, kl - j0, D, vec);
    load_rows<T, DP>(sV, v + (int64_t)j0 * a.sv.t, a.sv.t, kl - j0, D, vec);
    __syncthreads();
    float s[4][4] = {};
    dot_tile<DP>(sQ, sK, ty, tx, s);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int il = 4 * ty + x;
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int j = j0 + tx + 16 * c;
        const unsigned r = (unsigned)(j - (i0 + il + off) + a.window);
        const bool near = r < (unsigned)a.nrel, ok = j < n[x];
        if (near) s[x][c] += sR[r * kBT + il];
        s[x][c] = ok ? s[x][c] * sl2 : -INFINITY;
        if (near) sR[r * kBT + il] = s[x][c];
        mx = fmaxf(mx, s[x][c]);
      }
      mx = fmaxf(m[x], row_max(mx));
      const float mu = mx == -INFINITY ? 0.f : mx;
      const float alpha = exp2f(m[x] - mu);
      m[x] = mx;
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float p = exp2f(s[x][c] - mu);
        sP[(tx + 16 * c) * kLdP + il] = p;
        sum += p;
      }
      l[x] = l[x] * alpha + row_sum(sum);
#pragma unroll
      for (int w = 0; w < W; ++w) acc[x][w] *= alpha;
    }
    __syncthreads();
    acc_tile<DP>(sP, sV, ty, tx, acc);
  }
  __syncthreads();
  T* o = static_cast<T*>(a.o) + b * a.so.b + h * a.so.h;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int i = i0 + 4 * ty + x;
    if (i >= a.Tq) continue;
    const float mu = m[x] == -INFINITY ? 0.f : m[x];
    for (int r = 0; r < a.nrel; ++r) {
      const int j = i + off + r - a.window;
      if (j < 0 || j >= n[x]) continue;
      const float p = exp2f(sR[r * kBT + 4 * ty + x] - mu);
#pragma unroll
      for (int w = 0; w < W; ++w)
        if (tx * W + w < D) acc[x][w] = fmaf(p, to_f(relv[(int64_t)r * D + tx * W + w]), acc[x][w]);
    }
    const float inv = l[x] == 0.f ? 0.f : 1.f / l[x];
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (tx * W + w < D) o[(int64_t)i * a.so.t + tx * W + w] = from_f<T>(l[x] == 0.f ? 0.f : acc[x][w] * inv);
    if (tx == 0 && a.lse)
      a.lse[((int64_t)b * a.H + h) * a.Tq + i] = l[x] == 0.f ? -INFINITY : (mu + log2f(l[x])) * kLn2;
  }
}

// Blocks [0, nk) of x: dk, dv of one key tile and key head; the rest: dq of one
// query tile, once per query head (the z axis carries the batch).
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) attn_bwd_simt(const AttnArgs a, const BwdWs ws, const int nk,
                                                          const bool vec) {
  constexpr int W = DP / 16;
  extern __shared__ __align__(16) float sm[];
  float* s0 = sm;  // the resident pair, then the streamed pair
  float* s1 = s0 + tile_floats<DP>();
  float* s2 = s1 + tile_floats<DP>();
  float* s3 = s2 + tile_floats<DP>();
  float* sP = s3 + tile_floats<DP>();
  float* sS = sP + kBT * kLdP;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int b = blockIdx.z, D = a.D, g = a.H / a.Hkv;
  const int ql = clamp_len(a.qlen, b, a.Tq), kl = clamp_len(a.klen, b, a.Tk), off = kl - ql;
  const float sl2 = a.scale * kLog2e;
  const bool keys = (int)blockIdx.x < nk;
  if (keys) {
    const int hk = blockIdx.y;
    if (hk >= a.Hkv) return;
    const int j0 = blockIdx.x * kBT;
    load_rows<T, DP>(s0, static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h + (int64_t)j0 * a.sk.t, a.sk.t,
                     kl - j0, D, vec);
    load_rows<T, DP>(s1, static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h + (int64_t)j0 * a.sv.t, a.sv.t,
                     kl - j0, D, vec);
    float dk[4][W] = {}, dv[4][W] = {};
    const int first = j0 >= kl ? ql : (a.causal ? max(0, j0 - off) / kBT * kBT : 0);
    for (int hh = 0; hh < g; ++hh) {
      const int h = hk * g + hh;
      const int64_t bh = (int64_t)b * a.H + h;
      for (int i0 = first; i0 < ql; i0 += kBT) {
        __syncthreads();
        load_rows<T, DP>(s2, static_cast<const T*>(a.q) + b * a.sq.b + h * a.sq.h + (int64_t)i0 * a.sq.t, a.sq.t,
                         ql - i0, D, vec);
        load_rows<T, DP>(s3, static_cast<const T*>(a.dout) + b * a.sdo.b + h * a.sdo.h + (int64_t)i0 * a.sdo.t,
                         a.sdo.t, ql - i0, D, vec);
        __syncthreads();
        float s[4][4] = {}, dp[4][4] = {};
        dot_tile<DP>(s0, s2, ty, tx, s);
        dot_tile<DP>(s1, s3, ty, tx, dp);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int i = i0 + tx + 16 * c;
          const int n = allowed_keys(i, ql, kl, a.causal);
          const float* rw = row_at(ws, bh, i);
          const float nlse2 = n > 0 ? rw[0] : 0.f, ndelta = n > 0 ? rw[kRowBlock] : 0.f;
          const float* qr = rel_at(ws, bh, i, a.nrel);
          float p4[4], s4[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int j = j0 + 4 * ty + x;
            const unsigned r = (unsigned)(j - (i + off) + a.window);
            const bool ok = j < n;
            if (ok && r < (unsigned)a.nrel) {
              s[x][c] += qr[r];
              dp[x][c] += qr[kRowBlock * a.nrel + r];
            }
            p4[x] = ok ? exp2f(fmaf(s[x][c], sl2, nlse2)) : 0.f;
            s4[x] = ok ? p4[x] * (dp[x][c] + ndelta) : 0.f;
          }
          *reinterpret_cast<float4*>(sP + (tx + 16 * c) * kLdP + 4 * ty) = make_float4(p4[0], p4[1], p4[2], p4[3]);
          *reinterpret_cast<float4*>(sS + (tx + 16 * c) * kLdP + 4 * ty) = make_float4(s4[0], s4[1], s4[2], s4[3]);
        }
        __syncthreads();
        acc_tile<DP>(sP, s3, ty, tx, dv);
        acc_tile<DP>(sS, s2, ty, tx, dk);
      }
    }
    T* odk = static_cast<T*>(a.dk) + b * a.sdk.b + hk * a.sdk.h;
    T* odv = static_cast<T*>(a.dv) + b * a.sdv.b + hk * a.sdv.h;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int j = j0 + 4 * ty + x;
      if (j >= a.Tk) continue;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (tx * W + w >= D) continue;
        odk[(int64_t)j * a.sdk.t + tx * W + w] = from_f<T>(dk[x][w] * a.scale);
        odv[(int64_t)j * a.sdv.t + tx * W + w] = from_f<T>(dv[x][w]);
      }
    }
    return;
  }
  const int h = blockIdx.y, hk = h / g;
  const int i0 = (blockIdx.x - nk) * kBT;
  const int64_t bh = (int64_t)b * a.H + h, row = bh * a.Tq;
  load_rows<T, DP>(s0, static_cast<const T*>(a.q) + b * a.sq.b + h * a.sq.h + (int64_t)i0 * a.sq.t, a.sq.t, ql - i0,
                   D, vec);
  load_rows<T, DP>(s1, static_cast<const T*>(a.dout) + b * a.sdo.b + h * a.sdo.h + (int64_t)i0 * a.sdo.t, a.sdo.t,
                   ql - i0, D, vec);
  float dq[4][W] = {}, nlse2[4], ndelta[4];
  int n[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int i = i0 + 4 * ty + x;
    n[x] = allowed_keys(i, ql, kl, a.causal);
    const float* rw = row_at(ws, bh, i);
    nlse2[x] = n[x] > 0 ? rw[0] : 0.f;
    ndelta[x] = n[x] > 0 ? rw[kRowBlock] : 0.f;
  }
  const int last = min(i0 + kBT, ql) - 1;
  const int kend = last < i0 ? 0 : allowed_keys(last, ql, kl, a.causal);
  for (int j0 = 0; j0 < kend; j0 += kBT) {
    __syncthreads();
    load_rows<T, DP>(s2, static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h + (int64_t)j0 * a.sk.t, a.sk.t,
                     kl - j0, D, vec);
    load_rows<T, DP>(s3, static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h + (int64_t)j0 * a.sv.t, a.sv.t,
                     kl - j0, D, vec);
    __syncthreads();
    float s[4][4] = {}, dp[4][4] = {};
    dot_tile<DP>(s0, s2, ty, tx, s);
    dot_tile<DP>(s1, s3, ty, tx, dp);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int j = j0 + tx + 16 * c;
      float s4[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int i = i0 + 4 * ty + x;
        const unsigned r = (unsigned)(j - (i + off) + a.window);
        const bool ok = j < n[x], near = ok && r < (unsigned)a.nrel;
        if (near) {
          const float* qr = rel_at(ws, bh, i, a.nrel);
          s[x][c] += qr[r];
          dp[x][c] += qr[kRowBlock * a.nrel + r];
        }
        const float p = ok ? exp2f(fmaf(s[x][c], sl2, nlse2[x])) : 0.f;
        s4[x] = ok ? p * (dp[x][c] + ndelta[x]) : 0.f;
        if (near) {
          ws.pband[(row + i) * a.nrel + r] = p;
          ws.sband[(row + i) * a.nrel + r] = s4[x];
        }
      }
      *reinterpret_cast<float4*>(sS + (tx + 16 * c) * kLdP + 4 * ty) = make_float4(s4[0], s4[1], s4[2], s4[3]);
    }
    __syncthreads();
    acc_tile<DP>(sS, s2, ty, tx, dq);
  }
  __syncthreads();  // the near terms written by other threads of the block
  const T* relk = static_cast<const T*>(a.relk);
  T* o = static_cast<T*>(a.dq) + b * a.sdq.b + h * a.sdq.h;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int i = i0 + 4 * ty + x;
    if (i >= a.Tq) continue;
    for (int r = 0; r < a.nrel; ++r) {
      const int j = i + off + r - a.window;
      if (j < 0 || j >= n[x]) continue;
      const float ds = ws.sband[(row + i) * a.nrel + r];
#pragma unroll
      for (int w = 0; w < W; ++w)
        if (tx * W + w < D) dq[x][w] = fmaf(ds, to_f(relk[(int64_t)r * D + tx * W + w]), dq[x][w]);
    }
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (tx * W + w < D) o[(int64_t)i * a.sdq.t + tx * W + w] = from_f<T>(dq[x][w] * a.scale);
  }
}

template <typename T, int DP>
cudaError_t fwd(const AttnArgs& a, cudaStream_t st) {
  const size_t smem = sizeof(float) * (3 * tile_floats<DP>() + kBT * kLdP + a.nrel * kBT);
  cudaError_t e = cudaFuncSetAttribute(attn_fwd_simt<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const int el = sizeof(T);
  const bool vec = attn_rows_aligned(a.q, a.sq, a.D, el) && attn_rows_aligned(a.k, a.sk, a.D, el) &&
                   attn_rows_aligned(a.v, a.sv, a.D, el);
  attn_fwd_simt<T, DP><<<dim3(cdiv(a.Tq, kBT), a.H, a.B), kThreads, smem, st>>>(a, vec);
  return cudaGetLastError();
}

template <typename T, int DP>
cudaError_t bwd(const AttnArgs& a, const BwdWs& ws, cudaStream_t st) {
  const size_t smem = sizeof(float) * (4 * tile_floats<DP>() + 2 * kBT * kLdP);
  cudaError_t e = cudaFuncSetAttribute(attn_bwd_simt<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  const int el = sizeof(T);
  const bool vec = attn_rows_aligned(a.q, a.sq, a.D, el) && attn_rows_aligned(a.k, a.sk, a.D, el) &&
                   attn_rows_aligned(a.v, a.sv, a.D, el) && attn_rows_aligned(a.dout, a.sdo, a.D, el);
  const int nk = cdiv(a.Tk, kBT), nq = cdiv(a.Tq, kBT);
  attn_bwd_simt<T, DP><<<dim3(nk + nq, a.H, a.B), kThreads, smem, st>>>(a, ws, nk, vec);
  return cudaGetLastError();
}

template <typename T>
cudaError_t fwd_d(const AttnArgs& a, cudaStream_t st) {
  if (a.D <= 32) return fwd<T, 32>(a, st);
  if (a.D <= 64) return fwd<T, 64>(a, st);
  if (a.D <= 96) return fwd<T, 96>(a, st);
  return fwd<T, 128>(a, st);
}
template <typename T>
cudaError_t bwd_d(const AttnArgs& a, const BwdWs& ws, cudaStream_t st) {
  if (a.D <= 32) return bwd<T, 32>(a, ws, st);
  if (a.D <= 64) return bwd<T, 64>(a, ws, st);
  if (a.D <= 96) return bwd<T, 96>(a, ws, st);
  return bwd<T, 128>(a, ws, st);
}

}  // namespace

cudaError_t attn_fwd_cores(const AttnArgs& a, cudaStream_t st) {
  return fwd_d<float>(a, st);
}

cudaError_t attn_bwd_cores(const AttnArgs& a, const BwdWs& ws, cudaStream_t st) {
  return bwd_d<float>(a, ws, st);
}

}  // namespace gsv
