// norm_grad.cu -- residual LayerNorm forward with its statistics, and its
// backward with the reduction of the weight gradients (formulas in
// norm_grad.h).
//
// Both directions are bound by HBM: the forward reads x, y and writes out, the
// backward reads x, y, dout and writes dx, each element once.  Every element
// stays in registers between its load and its store; mean and variance are
// two sums over those registers (no cancellation, no second read).
//
// [B][T][C]: R threads of a block (a power of two, 32 .. 256) share one frame
// and hold up to E channels each as 16-byte vectors; a frame's sums go through
// shuffles and, for R > 32, shared memory.  Rows that do not start on 16-byte
// boundaries take single elements instead (V = 1), lanes side by side.
// [B][C][T]: a block takes 32 frames, one per lane, and its 16 warps up to E
// channels each; more than 16 E channels are split over a cluster whose blocks
// exchange the frame sums through distributed shared memory.
//
// The backward's blocks walk many frames and keep dgamma / dbeta of their
// channels in fp32 registers, written once per block as partial sums that a
// second kernel adds in block order: no atomics, so the result does not depend
// on scheduling.
#include <cooperative_groups.h>

#include <algorithm>

#include "attn_common.cuh"
#include "norm_grad.h"

namespace cg = cooperative_groups;

namespace gsv {
namespace {

constexpr int kRowThreads = 256;
constexpr int kTimeWarps = 16;
constexpr int kTimeE = 16;  // channels per thread, largest: 256 channels per block

template <typename T, int V>
struct Vec {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float* f) {
  if constexpr (V == 1) {
    f[0] = to_f(*p);
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f(e[i]);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float* f) {
  if constexpr (V == 1) {
    *p = from_f<T>(f[0]);
  } else {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_f<T>(f[i]);
    *reinterpret_cast<uint4*>(p) = u;
  }
}

// Sum of NS values over the R threads of a frame group; every thread gets it.
// All threads of the block call it together.
template <int R, int NS>
__device__ __forceinline__ void group_sum(float* v, float* s_red) {
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  if constexpr (R > 32) {
    const int w = threadIdx.x >> 5, g = threadIdx.x / R, nw = R / 32;
    __syncthreads();  // the previous use has been read
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int n = 0; n < NS; ++n) s_red[w * NS + n] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      v[n] = 0.f;
      for (int k = 0; k < nw; ++k) v[n] += s_red[(g * nw + k) * NS + n];
    }
  }
}

template <typename T, int V, int E, int R>
__global__ void __launch_bounds__(kRowThreads) norm_fwd_rows(const NormArgs a) {
  constexpr int N = E / V, G = kRowThreads / R;
  __shared__ float s_red[8];
  const int tid = threadIdx.x % R, grp = threadIdx.x / R, C = a.C;
  const int64_t frames = (int64_t)a.B * a.T;
  const int64_t f = (int64_t)blockIdx.x * G + grp;
  const bool in = f < frames;
  const int b = in ? (int)(f / a.T) : 0, t = in ? (int)(f - (int64_t)b * a.T) : 0;
  const bool ok = in && (!a.len || t < a.len[b]);
  const T* x = static_cast<const T*>(a.x.p) + b * a.x.b + t * a.x.o;
  const T* y = static_cast<const T*>(a.y.p) + b * a.y.b + t * a.y.o;
  float s[E] = {}, u[E] = {};
  if (ok) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int c = (tid + k * R) * V;
      if (c < C) load_vec<T, V>(x + c, s + k * V);
    }
    if (a.y.p) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int c = (tid + k * R) * V;
        if (c < C) load_vec<T, V>(y + c, u + k * V);
      }
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    s[e] += u[e];
    sum += s[e];
  }
  group_sum<R, 1>(&sum, s_red);
  const float mean = sum / (float)C;
  float sq = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k)
    if ((tid + k * R) * V < C)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = s[k * V + i] - mean;
        sq = fmaf(d, d, sq);
      }
  group_sum<R, 1>(&sq, s_red);
  const float rstd = rsqrtf(sq / (float)C + a.eps);
  if (!in) return;
  if (tid == 0) {
    a.mean[f] = ok ? mean : 0.f;
    a.rstd[f] = ok ? rstd : 0.f;
  }
  T* out = static_cast<T*>(const_cast<void*>(a.out.p)) + b * a.out.b + t * a.out.o;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int c = (tid + k * R) * V;
    if (c >= C) continue;
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = ok ? fmaf((s[k * V + i] - mean) * rstd, a.gamma[c + i], a.beta[c + i]) : 0.f;
    store_vec<T, V>(out + c, o);
  }
}

template <typename T, int V, int E, int R>
__global__ void __launch_bounds__(kRowThreads) norm_bwd_rows(const NormArgs a) {
  constexpr int N = E / V, G = kRowThreads / R;
  extern __shared__ float s_part[];  // [2][C] when several groups share the block's partial sums
  __shared__ float s_red[16];
  const int tid = threadIdx.x % R, grp = threadIdx.x / R, C = a.C;
  const int64_t frames = (int64_t)a.B * a.T;
  float dg[E] = {}, db[E] = {}, ga[E] = {};
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int c = (tid + k * R) * V;
    if (c < C)
#pragma unroll
      for (int i = 0; i < V; ++i) ga[k * V + i] = a.gamma[c + i];
  }
  // Every thread of the block runs the same number of steps (block barriers inside).
  for (int64_t f0 = (int64_t)blockIdx.x * G; f0 < frames; f0 += (int64_t)gridDim.x * G) {
    const int64_t f = f0 + grp;
    const bool in = f < frames;
    const int b = in ? (int)(f / a.T) : 0, t = in ? (int)(f - (int64_t)b * a.T) : 0;
    const bool ok = in && (!a.len || t < a.len[b]);
    float xh[E] = {}, g[E] = {}, sums[2] = {0.f, 0.f};
    float rstd = 0.f;
    if (ok) {
      const T* x = static_cast<const T*>(a.x.p) + b * a.x.b + t * a.x.o;
      const T* y = static_cast<const T*>(a.y.p) + b * a.y.b + t * a.y.o;
      const T* go = static_cast<const T*>(a.dout.p) + b * a.dout.b + t * a.dout.o;
      float u[E] = {};
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int c = (tid + k * R) * V;
        if (c < C) {
          load_vec<T, V>(x + c, xh + k * V);
          load_vec<T, V>(go + c, g + k * V);
          if (a.y.p) load_vec<T, V>(y + c, u + k * V);
        }
      }
      const float mean = a.mean[f];
      rstd = a.rstd[f];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if ((tid + k * R) * V >= C) continue;
#pragma unroll
        for (int e = k * V; e < (k + 1) * V; ++e) {
          xh[e] = (xh[e] + u[e] - mean) * rstd;
          dg[e] = fmaf(g[e], xh[e], dg[e]);
          db[e] += g[e];
          g[e] *= ga[e];
          sums[0] += g[e];
          sums[1] = fmaf(g[e], xh[e], sums[1]);
        }
      }
    }
    group_sum<R, 2>(sums, s_red);
    const float m0 = sums[0] / (float)C, m1 = sums[1] / (float)C;
    if (!in) continue;
    T* dx = static_cast<T*>(const_cast<void*>(a.dx.p)) + b * a.dx.b + t * a.dx.o;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int c = (tid + k * R) * V;
      if (c >= C) continue;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = rstd * (g[k * V + i] - m0 - xh[k * V + i] * m1);
      store_vec<T, V>(dx + c, o);
    }
  }
  float* part = a.part + (int64_t)blockIdx.x * 2 * C;
  // The groups add their sums in turn, so the order is fixed.
  for (int w = 0; w < G; ++w) {
    if (grp == w) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int c = (tid + k * R) * V;
        if (c >= C) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (w > 0) {
            dg[k * V + i] += s_part[c + i];
            db[k * V + i] += s_part[C + c + i];
          }
          if (w < G - 1) {
            s_part[c + i] = dg[k * V + i];
            s_part[C + c + i] = db[k * V + i];
          } else {
            part[c + i] = dg[k * V + i];
            part[C + c + i] = db[k * V + i];
          }
        }
      }
    }
    __syncthreads();
  }
}

// Sums of NS values per frame (lane) over the block's warps and the cluster.
template <int NS>
__device__ __forceinline__ void frame_sum(float* v, float (*s_w)[NS][32], float (*s_b)[32], cg::cluster_group& cl,
                                          int cs) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int n = 0; n < NS; ++n) s_w[w][n][lane] = v[n];
  __syncthreads();
  if (cs == 1) {
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      v[n] = 0.f;
#pragma unroll
      for (int k = 0; k < kTimeWarps; ++k) v[n] += s_w[k][n][lane];
    }
    __syncthreads();
    return;
  }
  if (w < NS) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < kTimeWarps; ++k) t += s_w[k][w][lane];
    s_b[w][lane] = t;
  }
  cl.sync();
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    v[n] = 0.f;
    for (int k = 0; k < cs; ++k) v[n] += *cl.map_shared_rank(&s_b[n][lane], k);
  }
  cl.sync();  // the sums have been read by every block
}

// blockIdx.x = (tile, cluster rank); a tile is 32 frames of one utterance.
template <typename T, int E>
__global__ void __launch_bounds__(kTimeWarps * 32) norm_fwd_time(const NormArgs a, const int cs) {
  __shared__ float s_w[kTimeWarps][1][32];
  __shared__ float s_b[1][32];
  cg::cluster_group cl = cg::this_cluster();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, C = a.C;
  const int tiles = cdiv(a.T, 32), tile = blockIdx.x / cs, rank = blockIdx.x - tile * cs;
  const int b = tile / tiles, t = (tile - b * tiles) * 32 + lane;
  const bool in = t < a.T, ok = in && (!a.len || t < a.len[b]);
  const int c0 = rank * kTimeWarps * E + w;
  const T* x = static_cast<const T*>(a.x.p) + b * a.x.b + t;
  const T* y = static_cast<const T*>(a.y.p) + b * a.y.b + t;
  float s[E] = {}, u[E] = {};
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = c0 + e * kTimeWarps;
    if (ok && c < C) {
      s[e] = to_f(x[c * a.x.o]);
      if (a.y.p) u[e] = to_f(y[c * a.y.o]);
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    s[e] += u[e];
    sum += s[e];
  }
  frame_sum<1>(&sum, s_w, s_b, cl, cs);
  const float mean = sum / (float)C;
  float sq = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (c0 + e * kTimeWarps < C) sq = fmaf(s[e] - mean, s[e] - mean, sq);
  frame_sum<1>(&sq, s_w, s_b, cl, cs);
  const float rstd = rsqrtf(sq / (float)C + a.eps);
  if (!in) return;
  if (w == 0 && rank == 0) {
    a.mean[(int64_t)b * a.T + t] = ok ? mean : 0.f;
    a.rstd[(int64_t)b * a.T + t] = ok ? rstd : 0.f;
  }
  T* out = static_cast<T*>(const_cast<void*>(a.out.p)) + b * a.out.b + t;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = c0 + e * kTimeWarps;
    if (c < C) out[c * a.out.o] = from_f<T>(ok ? fmaf((s[e] - mean) * rstd, a.gamma[c], a.beta[c]) : 0.f);
  }
}

template <typename T, int E>
__global__ void __launch_bounds__(kTimeWarps * 32) norm_bwd_time(const NormArgs a, const int cs) {
  __shared__ float s_w[kTimeWarps][2][32];
  __shared__ float s_b[2][32];
  cg::cluster_group cl = cg::this_cluster();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, C = a.C;
  const int per_b = cdiv(a.T, 32), tiles = per_b * a.B, team = blockIdx.x / cs, rank = blockIdx.x - team * cs;
  const int teams = gridDim.x / cs;
  const int c0 = rank * kTimeWarps * E + w;
  float dg[E] = {}, db[E] = {};
  for (int tile = team; tile < tiles; tile += teams) {
    const int b = tile / per_b, t = (tile - b * per_b) * 32 + lane;
    const bool in = t < a.T, ok = in && (!a.len || t < a.len[b]);
    const T* x = static_cast<const T*>(a.x.p) + b * a.x.b + t;
    const T* y = static_cast<const T*>(a.y.p) + b * a.y.b + t;
    const T* go = static_cast<const T*>(a.dout.p) + b * a.dout.b + t;
    float xh[E] = {}, g[E] = {}, sums[2] = {0.f, 0.f}, mean = 0.f, rstd = 0.f;
    if (ok) {
      mean = a.mean[(int64_t)b * a.T + t];
      rstd = a.rstd[(int64_t)b * a.T + t];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = c0 + e * kTimeWarps;
      if (ok && c < C) {
        xh[e] = to_f(x[c * a.x.o]);
        g[e] = to_f(go[c * a.dout.o]);
      }
    }
    if (a.y.p) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = c0 + e * kTimeWarps;
        if (ok && c < C) xh[e] += to_f(y[c * a.y.o]);
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = c0 + e * kTimeWarps;
      if (c >= C) continue;
      xh[e] = (xh[e] - mean) * rstd;
      dg[e] = fmaf(g[e], xh[e], dg[e]);
      db[e] += g[e];
      g[e] *= a.gamma[c];
      sums[0] += g[e];
      sums[1] = fmaf(g[e], xh[e], sums[1]);
    }
    frame_sum<2>(sums, s_w, s_b, cl, cs);
    const float m0 = sums[0] / (float)C, m1 = sums[1] / (float)C;
    T* dx = static_cast<T*>(const_cast<void*>(a.dx.p)) + b * a.dx.b + t;
    if (in) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = c0 + e * kTimeWarps;
        if (c < C) dx[c * a.dx.o] = from_f<T>(rstd * (g[e] - m0 - xh[e] * m1));
      }
    }
  }
  float* part = a.part + (int64_t)team * 2 * C;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = c0 + e * kTimeWarps;
    if (c >= C) continue;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      dg[e] += __shfl_xor_sync(0xffffffffu, dg[e], o);
      db[e] += __shfl_xor_sync(0xffffffffu, db[e], o);
    }
    if (lane == 0) {
      part[c] = dg[e];
      part[C + c] = db[e];
    }
  }
}

// dgamma, dbeta = the partial sums added in block order: 32 columns per block,
// 8 runs of blocks side by side, then the 8 runs in turn.
__global__ void __launch_bounds__(256) norm_part_sum(const float* part, int blocks, int C, float* dgamma,
                                                     float* dbeta) {
  __shared__ float s[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int e = blockIdx.x * 32 + lane, n = 2 * C;
  float v = 0.f;
  if (e < n)
    for (int k = w; k < blocks; k += 8) v += part[(int64_t)k * n + e];
  s[w][lane] = v;
  __syncthreads();
  if (w == 0 && e < n) {
    for (int k = 1; k < 8; ++k) v += s[k][lane];
    if (e < C) dgamma[e] = v;
    else dbeta[e - C] = v;
  }
}

// Threads of a block that share a frame, and channels per thread: as few
// threads as hold the frame with 16 channels each, 256 threads with 32 beyond.
struct RowShape {
  int R, E;
};
RowShape row_shape(int C) {
  if (C <= 256) return {32, 8};
  if (C <= 512) return {32, 16};
  if (C <= 1024) return {64, 16};
  if (C <= 2048) return {128, 16};
  if (C <= 4096) return {256, 16};
  return {256, 32};
}

int row_bwd_blocks(const NormArgs& a) {
  const RowShape s = row_shape(a.C);
  const int64_t n = ((int64_t)a.B * a.T + kRowThreads / s.R - 1) / (kRowThreads / s.R);
  return (int)std::max<int64_t>(1, std::min<int64_t>(n, 148 * 4));  // one block writes the zeros of no frames
}

int time_cluster(int C) {
  int cs = 1;
  while (cs * kTimeWarps * kTimeE < C) cs *= 2;
  return cs;
}

int time_bwd_teams(const NormArgs& a) {
  const int cs = time_cluster(a.C);
  return (int)std::max<int64_t>(1, std::min<int64_t>((int64_t)a.B * cdiv(a.T, 32), 148 * 2 / cs));
}

bool vec_ok(const NormTensor& t, int C, int V, int elem) {
  return !t.p || (reinterpret_cast<uintptr_t>(t.p) % 16 == 0 && t.b % V == 0 && t.o % V == 0 && C % V == 0 &&
                  16 / elem == V);
}

template <typename T, int V, int E, int R>
cudaError_t rows_launch(const NormArgs& a, bool bwd, cudaStream_t st) {
  constexpr int G = kRowThreads / R;
  if (!bwd) {
    const int64_t n = ((int64_t)a.B * a.T + G - 1) / G;
    norm_fwd_rows<T, V, E, R><<<(unsigned)n, kRowThreads, 0, st>>>(a);
  } else {
    const size_t smem = G > 1 ? 2 * (size_t)a.C * sizeof(float) : 0;
    norm_bwd_rows<T, V, E, R><<<row_bwd_blocks(a), kRowThreads, smem, st>>>(a);
  }
  return cudaGetLastError();
}

template <typename T, int V>
cudaError_t rows_shape(const NormArgs& a, bool bwd, cudaStream_t st) {
  const RowShape s = row_shape(a.C);
  if (s.R == 32) return s.E == 8 ? rows_launch<T, V, 8, 32>(a, bwd, st) : rows_launch<T, V, 16, 32>(a, bwd, st);
  if (s.R == 64) return rows_launch<T, V, 16, 64>(a, bwd, st);
  if (s.R == 128) return rows_launch<T, V, 16, 128>(a, bwd, st);
  return s.E == 16 ? rows_launch<T, V, 16, 256>(a, bwd, st) : rows_launch<T, V, 32, 256>(a, bwd, st);
}

template <typename T, int E>
cudaError_t time_launch(const NormArgs& a, bool bwd, int cs, cudaStream_t st) {
  const int64_t tiles = (int64_t)a.B * cdiv(a.T, 32);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((bwd ? time_bwd_teams(a) : tiles) * cs));
  cfg.blockDim = dim3(kTimeWarps * 32);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cs;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return bwd ? cudaLaunchKernelEx(&cfg, norm_bwd_time<T, E>, a, cs) : cudaLaunchKernelEx(&cfg, norm_fwd_time<T, E>, a, cs);
}

template <typename T>
cudaError_t run_t(const NormArgs& a, bool bwd, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  if (a.rows) {
    const bool vec = vec_ok(a.x, a.C, V, sizeof(T)) && vec_ok(a.y, a.C, V, sizeof(T)) &&
                     (bwd ? vec_ok(a.dout, a.C, V, sizeof(T)) && vec_ok(a.dx, a.C, V, sizeof(T))
                          : vec_ok(a.out, a.C, V, sizeof(T)));
    return vec ? rows_shape<T, V>(a, bwd, st) : rows_shape<T, 1>(a, bwd, st);
  }
  const int cs = time_cluster(a.C), e = cdiv(cdiv(a.C, cs), kTimeWarps);
  // With several blocks per frame each takes its full 256 channels.
  if (cs > 1 || e > 12) return time_launch<T, 16>(a, bwd, cs, st);
  if (e > 8) return time_launch<T, 12>(a, bwd, cs, st);
  return e > 4 ? time_launch<T, 8>(a, bwd, cs, st) : time_launch<T, 4>(a, bwd, cs, st);
}

cudaError_t run(const NormArgs& a, bool bwd, cudaStream_t st) {
  switch (a.ty) {
    case Ty::F32: return run_t<float>(a, bwd, st);
    case Ty::F16: return run_t<__half>(a, bwd, st);
    default: return run_t<__nv_bfloat16>(a, bwd, st);
  }
}

}  // namespace

size_t norm_bwd_workspace(const NormArgs& a) {
  const int n = a.rows ? row_bwd_blocks(a) : time_bwd_teams(a);
  return (size_t)n * 2 * a.C * sizeof(float);
}

cudaError_t norm_forward(const NormArgs& a, cudaStream_t st) { return a.T ? run(a, false, st) : cudaSuccess; }

cudaError_t norm_backward(const NormArgs& a, cudaStream_t st) {
  const cudaError_t e = run(a, true, st);
  if (e != cudaSuccess) return e;
  const int n = a.rows ? row_bwd_blocks(a) : time_bwd_teams(a);
  norm_part_sum<<<cdiv(2 * a.C, 32), 256, 0, st>>>(a.part, n, a.C, a.dgamma, a.dbeta);
  return cudaGetLastError();
}

}  // namespace gsv
