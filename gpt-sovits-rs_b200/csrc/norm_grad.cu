// norm_grad.cu -- residual LayerNorm forward with its statistics, and its
// backward with the reduction of the weight gradients (formulas in
// norm_grad.h).
//
// Both directions are bound by HBM: the forward reads x, y and writes out, the
// backward reads x, y, dout and writes dx, each element once.  Every element
// stays in registers between its load and its store; mean and variance are
// two sums over those registers (no cancellation, no second read).
//
// [B][T][C]: R threads (a power of two, 32 .. 256) share one frame and hold up
// to E channels each.  Blocks are persistent; every group of R threads has a
// ring of frames in shared memory that one lane fills by bulk copies, so that
// the loads of the next frames are in flight whatever the registers do.  Rows
// that are not whole aligned 16-byte vectors (V = 1) are loaded directly.
// [B][C][T]: a block takes 32 frames; a lane holds V of them (4 where rows are
// aligned for vectors of 4, else 1) for up to 16 / V channels per warp and
// lane.  More than 256 channels are split over a cluster whose blocks exchange
// the frame sums through distributed shared memory.
//
// The backward's blocks walk many frames and keep dgamma / dbeta of their
// channels in fp32 registers, written once per block as partial sums that a
// second kernel adds in block order: no atomics, so the result does not depend
// on scheduling.
//
// Measured on B200, bf16 [8][4096][1024]: forward 37 us, 5.4 TB/s (83 % of a
// copy's bandwidth; 69 us where rows are not aligned, here of 1023), backward
// 60 us, 4.5 TB/s (80 unaligned): it waits for fixed latencies, the barrier of
// each frame and shared memory (issue slots 56 %), hardly for HBM.  fp32
// [8][2048][1024]: 37.7 and 50.3 us, 82 % of a copy's bandwidth both.  [B][C][T],
// fp32 [64][192][500]: forward 15.8 us, backward 20.5 with ragged lengths, 4 of
// them the second kernel; in single frames (T = 501) 18.2 and 31.6.  One
// sentence, [1][192][37]: 5.6 us, launch and two barriers.
#include <cooperative_groups.h>

#include <algorithm>

#include "attn_tc.cuh"
#include "gsv_pdl.cuh"
#include "norm_grad.h"

namespace cg = cooperative_groups;

namespace gsv {
namespace {

__device__ int g_give_ups;  // bounded waits of the kernels below that ran out

constexpr int kRowThreads = 256;
constexpr int kTimeWarps = 16;
constexpr int kTimeC = 256;  // channels of one block

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float* f) {
  if constexpr (V == 1) {
    f[0] = to_f(*p);
  } else if constexpr (V * sizeof(T) == 8) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f(e[i]);
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
  } else if constexpr (V * sizeof(T) == 8) {
    uint2 u;
    u.x = pack2<T>(f[0], f[1]);
    u.y = pack2<T>(f[2], f[3]);
    *reinterpret_cast<uint2*>(p) = u;
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    uint4 u;
    u.x = pack2<T>(f[0], f[1]);
    u.y = pack2<T>(f[2], f[3]);
    u.z = pack2<T>(f[4], f[5]);
    u.w = pack2<T>(f[6], f[7]);
    *reinterpret_cast<uint4*>(p) = u;
  }
}

// Sums of NS values over the R threads of a group; every thread gets them.  The
// buffer alternates between two halves, so one barrier per use is enough.
template <int R, int NS>
__device__ __forceinline__ void group_sum(float* v, float* s_red, int& flip) {
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  if constexpr (R > 32) {
    constexpr int W = R / 32;
    const int grp = threadIdx.x / R, w = threadIdx.x % R / 32;
    float* buf = s_red + (flip * (kRowThreads / 32) + grp * W) * NS;
    flip ^= 1;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int n = 0; n < NS; ++n) buf[w * NS + n] = v[n];
    asm volatile("bar.sync %0, %1;" ::"r"(1 + grp), "n"(R) : "memory");
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      v[n] = 0.f;
#pragma unroll
      for (int k = 0; k < W; ++k) v[n] += buf[k * NS + n];
    }
  } else {
    __syncwarp();
  }
}

__device__ __forceinline__ void bulk_row(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

constexpr int kMaxStages = 8;

template <typename T, int V, int E, int R, bool BWD>
__global__ void __launch_bounds__(kRowThreads, BWD && E > 16 ? 1 : 2) norm_rows(const __grid_constant__ NormArgs a, const int stages) {
  constexpr int N = E / V, G = kRowThreads / R, K = BWD ? 3 : 2;
  constexpr bool kRing = V > 1;
  extern __shared__ __align__(16) uint8_t s_ring[];  // [G][stages][K][C] of T
  __shared__ float s_red[2 * (kRowThreads / 32) * 2];
  __shared__ __align__(8) uint64_t s_bar[G][kMaxStages];
  __shared__ int s_abort;
  const int tid = threadIdx.x % R, grp = threadIdx.x / R, C = a.C;
  const uint32_t row_bytes = (uint32_t)C * sizeof(T);
  const int frames = a.B * a.T, step = gridDim.x * G;
  int flip = 0;
  if (kRing) {
    if (tid == 0) {
      for (int s = 0; s < stages; ++s) mbar_init(smem_u32(&s_bar[grp][s]), 1);
      fence_async_smem();  // by the lane that wrote them: a fence orders its own thread's writes only
    }
    if (threadIdx.x == 0) s_abort = 0;
    __syncthreads();
  }
  float ga[E], be[E];  // backward: be accumulates dbeta, dg dgamma
  float dg[BWD ? E : 1] = {};
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (tid + k * R) * V + i;
      ga[k * V + i] = c < C ? a.gamma[c] : 0.f;
      be[k * V + i] = !BWD && c < C ? a.beta[c] : 0.f;
    }
  auto valid = [&](int f, int& b, int& t) {
    b = f / a.T;
    t = f - b * a.T;
    return f < frames && (!a.len || t < a.len[b]);
  };
  const T* X = static_cast<const T*>(a.x.p);
  const T* Y = static_cast<const T*>(a.y.p);
  const T* D = static_cast<const T*>(a.dout.p);
  const uint8_t* ring = s_ring + (size_t)grp * stages * K * row_bytes;
  auto fetch = [&](int f, int s) {  // one lane: frame f's rows into stage s
    int b, t;
    if (!valid(f, b, t)) return;
    const uint32_t bar = smem_u32(&s_bar[grp][s]), dst = smem_u32(ring + (size_t)s * K * row_bytes);
    mbar_expect_tx(bar, row_bytes * (1 + (Y ? 1 : 0) + (BWD ? 1 : 0)));
    bulk_row(dst, X + b * a.x.b + t * a.x.o, row_bytes, bar);
    if (Y) bulk_row(dst + row_bytes, Y + b * a.y.b + t * a.y.o, row_bytes, bar);
    if (BWD) bulk_row(dst + 2 * row_bytes, D + b * a.dout.b + t * a.dout.o, row_bytes, bar);
  };
  const int f0 = blockIdx.x * G + grp;
  if (kRing && tid == 0)
    for (int s = 0; s < stages; ++s)
      if (f0 + (int64_t)s * step < frames) fetch(f0 + s * step, s);
  int s = 0;
  uint32_t phases = 0;
  // The statistics of the next frame are on their way while this one is worked on.
  float mean_next = BWD && f0 < frames ? a.mean[f0] : 0.f, rstd_next = BWD && f0 < frames ? a.rstd[f0] : 0.f;
  for (int64_t ff = f0; ff < frames; ff += step) {
    const int f = (int)ff;
    int b, t;
    const bool ok = valid(f, b, t);
    float v[E], g[BWD ? E : 1];
    // Statistics behind a length may hold anything, as the frames do.
    const float mean = ok ? mean_next : 0.f;
    float rstd = ok ? rstd_next : 0.f;
    if (BWD && ff + step < frames) {
      mean_next = a.mean[f + step];
      rstd_next = a.rstd[f + step];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll
    for (int e = 0; e < (BWD ? E : 1); ++e) g[e] = 0.f;
    if (ok) {
      if (kRing) {
        if (!warp_wait(smem_u32(&s_bar[grp][s]), phases >> s & 1, &s_abort)) {
          // The group cannot go on together: leave the kernel's results undefined, but end it.
          *const_cast<volatile int*>(&s_abort) = 1;
          give_up(nullptr, &g_give_ups);
        }
        phases ^= 1u << s;
        const T* sx = reinterpret_cast<const T*>(ring + (size_t)s * K * row_bytes);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int c = (tid + k * R) * V;
          if (c < C) {
            load_vec<T, V>(sx + c, v + k * V);
            if (Y) {
              float u[V];
              load_vec<T, V>(sx + C + c, u);
#pragma unroll
              for (int i = 0; i < V; i += 2)
                add2(F2(v[k * V + i], v[k * V + i + (V > 1)]), F2(u[i], u[i + (V > 1)]))
                    .get(v[k * V + i], v[k * V + i + (V > 1)]);
            }
            if (BWD) load_vec<T, V>(sx + 2 * C + c, g + k * V);
          }
        }
      } else {
        float u[E];
        // Clamped addresses: no load stands under a branch, so all are in flight together.
        const T* x = X + b * a.x.b + t * a.x.o;
        const T* y = Y ? Y + b * a.y.b + t * a.y.o : x;
        const T* d = BWD ? D + b * a.dout.b + t * a.dout.o : x;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int c = min(tid + e * R, C - 1);
          v[e] = to_f(x[c]);
          u[e] = to_f(y[c]);
          if (BWD) g[e] = to_f(d[c]);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const bool in = tid + e * R < C;
          v[e] = in ? (Y ? v[e] + u[e] : v[e]) : 0.f;
          if (BWD) g[e] = in ? g[e] : 0.f;
        }
      }
    }
    // Channels past C hold zeros; g is zero there too, so only (v - mean) has to be kept out of sums.
    float sums[2] = {0.f, 0.f};
    if (!BWD) {
      F2 sa(0.f, 0.f), sb(0.f, 0.f);
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        sa = add2(sa, F2(v[e], v[e + 1]));
        sb = add2(sb, F2(v[e + 2], v[e + 3]));
      }
      add2(sa, sb).get(sums[0], sums[1]);
      sums[0] += sums[1];
      group_sum<R, 1>(sums, s_red, flip);
    } else {
      F2 s0(0.f, 0.f), s1(0.f, 0.f);
      const F2 nm(-mean, -mean), rs(rstd, rstd);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const int z = BWD ? e : 0, z1 = BWD ? e + 1 : 0;
        const F2 xh = mul2(add2(F2(v[e], v[e + 1]), nm), rs);
        F2 q(g[z], g[z1]);
        fma2(q, xh, F2(dg[z], dg[z1])).get(dg[z], dg[z1]);
        add2(F2(be[e], be[e + 1]), q).get(be[e], be[e + 1]);
        q = mul2(q, F2(ga[e], ga[e + 1]));
        s0 = add2(s0, q);
        s1 = fma2(q, xh, s1);
        xh.get(v[e], v[e + 1]);
        q.get(g[z], g[z1]);
      }
      float lo, hi;
      s0.get(lo, hi);
      sums[0] = lo + hi;
      s1.get(lo, hi);
      sums[1] = lo + hi;
      group_sum<R, 2>(sums, s_red, flip);
    }
    // Every thread of the group has read the stage: it takes the frame `stages` steps on.
    if (kRing) {
      if (tid == 0 && ff + (int64_t)stages * step < frames) fetch(f + stages * step, s);
      if (++s == stages) s = 0;
    }
    const float m0 = sums[0] / (float)C;
    T* out = static_cast<T*>(const_cast<void*>(BWD ? a.dx.p : a.out.p)) + b * (BWD ? a.dx.b : a.out.b) +
             t * (BWD ? a.dx.o : a.out.o);
    if (!BWD) {
      F2 sq(0.f, 0.f);
      const F2 nm(-m0, -m0);
#pragma unroll
      for (int k = 0; k < N; ++k)
        if ((tid + k * R) * V < C) {
          if constexpr (V > 1) {
#pragma unroll
            for (int e = k * V; e < (k + 1) * V; e += 2) {
              const F2 d = add2(F2(v[e], v[e + 1]), nm);
              sq = fma2(d, d, sq);
              d.get(v[e], v[e + 1]);
            }
          } else {
            v[k] -= m0;
            float lo, hi;
            sq.get(lo, hi);
            sq = F2(fmaf(v[k], v[k], lo), hi);
          }
        }
      float lo, hi;
      sq.get(lo, hi);
      lo += hi;
      group_sum<R, 1>(&lo, s_red, flip);
      rstd = rsqrtf(lo / (float)C + a.eps);
      if (tid == 0) {
        a.mean[f] = ok ? m0 : 0.f;
        a.rstd[f] = ok ? rstd : 0.f;
      }
    }
    const float m1 = sums[1] / (float)C;
    // Backward: rstd (g - m0 - v m1) with rstd = 0 on frames left out.
    const F2 rs(rstd, rstd), n0(-m0, -m0), n1(-m1, -m1);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int c = (tid + k * R) * V;
      if (c >= C) continue;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        const int e = k * V + i, e1 = e + (V > 1), i1 = i + (V > 1);
        if (BWD) {
          const int z = BWD ? e : 0, z1 = BWD ? e1 : 0;
          mul2(fma2(F2(v[e], v[e1]), n1, add2(F2(g[z], g[z1]), n0)), rs).get(o[i], o[i1]);
        } else {
          fma2(mul2(F2(v[e], v[e1]), rs), F2(ga[e], ga[e1]), F2(be[e], be[e1])).get(o[i], o[i1]);
          if (!ok) o[i] = o[i1] = 0.f;
        }
      }
      store_vec<T, V>(out + c, o);
    }
  }
  if (BWD) {
    // The groups add their sums in turn over the ring's memory, so the order is fixed.
    float* s_part = reinterpret_cast<float*>(s_ring);
    float* part = a.part + (int64_t)blockIdx.x * 2 * C;
    __syncthreads();
    for (int w = 0; w < G; ++w) {
      if (grp == w) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int c = (tid + e / V * R) * V + e % V;
          if (c >= C) continue;
          const float x = dg[BWD ? e : 0] + (w > 0 ? s_part[c] : 0.f), y = be[e] + (w > 0 ? s_part[C + c] : 0.f);
          float* to = w < G - 1 ? s_part : part;
          to[c] = x;
          to[C + c] = y;
        }
      }
      __syncthreads();
    }
  }
}

// Sums of NS values for each of a lane's V frames over the block's warps and
// the cluster (lanes that share frames are added first).  s_b must be another
// buffer than the call's before: the one cluster barrier of each call then also
// says that the buffer before it has been read.
template <int NS, int V>
__device__ __forceinline__ void frame_sum(float (*v)[V], float (*s_w)[NS][32], float (*s_b)[32],
                                          cg::cluster_group& cl, int cs) {
  constexpr int F = 32 / V;  // lanes per row of frames
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int o = F; o < 32; o <<= 1) v[n][i] += __shfl_xor_sync(0xffffffffu, v[n][i], o);
      if (lane < F) s_w[w][n][lane * V + i] = v[n][i];
    }
  __syncthreads();
  if (w < NS) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < kTimeWarps; ++k) t += s_w[k][w][lane];
    s_b[w][lane] = t;
  }
  if (cs == 1) __syncthreads();
  else cl.sync();
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) v[n][i] = 0.f;
  for (int k = 0; k < cs; ++k) {
    const float* from = cs == 1 ? &s_b[0][0] : cl.map_shared_rank(&s_b[0][0], k);
#pragma unroll
    for (int n = 0; n < NS; ++n)
#pragma unroll
      for (int i = 0; i < V; ++i) v[n][i] += from[n * 32 + (lane % F) * V + i];
  }
}

// Blocks of a team (a cluster of cs) walk tiles of 32 frames of one utterance;
// a team's block r holds the channels from r * 16 E V.
template <typename T, int V, int E, bool BWD>
__global__ void __launch_bounds__(kTimeWarps * 32, BWD && V == 1 && E > 4 ? 1 : 2) norm_time(const __grid_constant__ NormArgs a, const int cs) {
  constexpr int F = 32 / V, NS = BWD ? 2 : 1;
  __shared__ float s_w[kTimeWarps][NS][32];
  __shared__ float s_b[2][NS][32];
  cg::cluster_group cl = cg::this_cluster();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, C = a.C;
  const int per_b = cdiv(a.T, 32), tiles = per_b * a.B, team = blockIdx.x / cs, rank = blockIdx.x - team * cs;
  const int teams = gridDim.x / cs;
  // A warp's load covers V channels side by side (lanes / F) of 32 frames.
  constexpr int kStep = kTimeWarps * V;
  const int c0 = rank * E * kStep + w * V + lane / F, fl = (lane % F) * V;
  // A lane with single frames has up to 16 channels: their weights are read where they are used.
  constexpr bool kHeld = V > 1;
  float ga[kHeld ? E : 1], be[BWD || kHeld ? E : 1], dg[BWD ? E : 1] = {};
  if (BWD)
#pragma unroll
    for (int e = 0; e < E; ++e) be[BWD ? e : 0] = 0.f;
  if constexpr (kHeld) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = c0 + e * kStep;
      ga[e] = c < C ? a.gamma[c] : 0.f;
      if (!BWD) be[e] = c < C ? a.beta[c] : 0.f;
    }
  }
  auto gamma = [&](int e) { return kHeld ? ga[kHeld ? e : 0] : a.gamma[min(c0 + e * kStep, C - 1)]; };
  auto beta = [&](int e) { return kHeld ? be[BWD || kHeld ? e : 0] : a.beta[min(c0 + e * kStep, C - 1)]; };
  int flip = 0;
  const int nc = c0 < C ? min(E, (C - c0 + kStep - 1) / kStep) : 0;  // this lane's channels
  for (int tile = team; tile < tiles; tile += teams) {
    const int b = tile / per_b, t = (tile - b * per_b) * 32 + fl;
    const int n = a.len ? a.len[b] : a.T;
    const bool in = t < a.T;
    float v[E][V], g[BWD ? E : 1][V], u[E][V], mean[V], rstd[V];
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < V; ++i) v[e][i] = u[e][i] = g[BWD ? e : 0][i] = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) mean[i] = rstd[i] = 0.f;
    if (t - fl < n) {  // the tile has frames to read (the same for the whole block)
      // With single frames a thread has up to 48 loads: clamped addresses, values dropped below, so that
      // none stands under a branch of its own and all are under way together.
      const bool some = in && t < n;
      const int tc = V == 1 ? min(t, a.T - 1) : t, cc = V == 1 ? min(c0, C - 1) : c0;
      const T* x = static_cast<const T*>(a.x.p) + b * a.x.b + tc + cc * a.x.o;
      const T* y = static_cast<const T*>(a.y.p) + b * a.y.b + tc + cc * a.y.o;
      const T* d = static_cast<const T*>(a.dout.p) + b * a.dout.b + tc + cc * a.dout.o;
      const int last = max(nc - 1, 0);
      if (BWD && (V == 1 || some)) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          mean[i] = a.mean[(int64_t)b * a.T + tc + i];
          rstd[i] = a.rstd[(int64_t)b * a.T + tc + i];
        }
      }
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (V == 1 || (some && e < nc)) load_vec<T, V>(x + (V == 1 ? min(e, last) : e) * (kStep * a.x.o), v[e]);
      if (a.y.p) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (V == 1 || (some && e < nc)) load_vec<T, V>(y + (V == 1 ? min(e, last) : e) * (kStep * a.y.o), u[e]);
      }
      if (BWD) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (V == 1 || (some && e < nc)) load_vec<T, V>(d + (V == 1 ? min(e, last) : e) * (kStep * a.dout.o), g[BWD ? e : 0]);
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (BWD && t + i >= n) mean[i] = rstd[i] = 0.f;
    float sums[NS][V] = {};
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const bool ok = t + i < n && t < a.T && e < nc;  // a frame behind the length may hold anything
        v[e][i] = ok ? v[e][i] + u[e][i] : 0.f;
        if (BWD) {
          const int z = BWD ? e : 0;
          v[e][i] = ok ? (v[e][i] - mean[i]) * rstd[i] : 0.f;
          const float q = ok ? g[z][i] : 0.f;
          dg[z] = fmaf(q, v[e][i], dg[z]);
          be[z] += q;
          g[z][i] = q * gamma(e);
          sums[0][i] += g[z][i];
          sums[NS - 1][i] = fmaf(g[z][i], v[e][i], sums[NS - 1][i]);
        } else {
          sums[0][i] += v[e][i];
        }
      }
    frame_sum<NS, V>(sums, s_w, s_b[flip], cl, cs);
    flip ^= 1;
    const float ic = 1.f / (float)C;
    if (!BWD) {
      float sq[1][V] = {};
#pragma unroll
      for (int i = 0; i < V; ++i) mean[i] = sums[0][i] * ic;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e < nc)
#pragma unroll
          for (int i = 0; i < V; ++i) sq[0][i] = fmaf(v[e][i] - mean[i], v[e][i] - mean[i], sq[0][i]);
      __syncthreads();  // the first sums of the block's warps have been read
      frame_sum<1, V>(sq, reinterpret_cast<float(*)[1][32]>(&s_w[0][0][0]), s_b[flip], cl, cs);
      flip ^= 1;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const bool ok = t + i < n;
        rstd[i] = ok ? rsqrtf(sq[0][i] * ic + a.eps) : 0.f;
        mean[i] = ok ? mean[i] : 0.f;
      }
      if (w == 0 && rank == 0 && lane < F && in)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          a.mean[(int64_t)b * a.T + t + i] = mean[i];
          a.rstd[(int64_t)b * a.T + t + i] = rstd[i];
        }
    }
    if (in) {
      const int64_t so = BWD ? a.dx.o : a.out.o;
      T* out = static_cast<T*>(const_cast<void*>(BWD ? a.dx.p : a.out.p)) + b * (BWD ? a.dx.b : a.out.b) + t + c0 * so;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (e >= nc) continue;
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i)
          o[i] = BWD ? rstd[i] * (g[BWD ? e : 0][i] - sums[0][i] * ic - v[e][i] * (sums[NS - 1][i] * ic))
                     : t + i < n ? fmaf((v[e][i] - mean[i]) * rstd[i], gamma(e), beta(e)) : 0.f;
        store_vec<T, V>(out + e * (kStep * so), o);
      }
    }
    __syncthreads();  // the sums' buffers are free for the next tile
  }
  if (cs > 1) cl.sync();  // the last sums have been read
  if (BWD) {
    float* part = a.part + (int64_t)team * 2 * C;
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
      for (int o = 1; o < F; o <<= 1) {
        dg[BWD ? e : 0] += __shfl_xor_sync(0xffffffffu, dg[BWD ? e : 0], o);
        be[BWD ? e : 0] += __shfl_xor_sync(0xffffffffu, be[BWD ? e : 0], o);
      }
      if (lane % F == 0 && e < nc) {
        part[c0 + e * kStep] = dg[BWD ? e : 0];
        part[C + c0 + e * kStep] = be[BWD ? e : 0];
      }
    }
  }
}

// dgamma, dbeta = the partial sums added in block order: 32 columns per block,
// 16 runs of blocks side by side, then the runs in turn.
__global__ void __launch_bounds__(512) norm_part_sum(const float* part, int blocks, int C, float* dgamma,
                                                     float* dbeta) {
  __shared__ float s[16][32];
  pdl_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int e = blockIdx.x * 32 + lane, n = 2 * C;
  float v = 0.f;
  if (e < n) {
#pragma unroll 8
    for (int k = w; k < blocks; k += 16) v += part[(int64_t)k * n + e];
  }
  s[w][lane] = v;
  __syncthreads();
  if (w == 0 && e < n) {
#pragma unroll
    for (int k = 1; k < 16; ++k) v += s[k][lane];
    if (e < C) dgamma[e] = v;
    else dbeta[e - C] = v;
  }
}

// Threads that share a frame, and channels per thread.  The forward holds 32
// channels a thread (one warp per frame up to 1024), the backward 16, since it
// also holds gamma and two sums for each (bf16 [8][4096][1024] backward: 64
// threads of 16 channels 60 us, 128 of 8 in three blocks per SM 72, 32 of 32 in
// one block 69).
struct RowShape {
  int R, E;
};
RowShape row_shape(int C, bool bwd) {
  if (C <= 256) return {32, 8};
  if (C <= 512) return {32, 16};
  if (!bwd) return C <= 1024 ? RowShape{32, 32} : C <= 2048 ? RowShape{64, 32} : C <= 4096 ? RowShape{128, 32} : RowShape{256, 32};
  return C <= 1024 ? RowShape{64, 16} : C <= 2048 ? RowShape{128, 16} : C <= 4096 ? RowShape{256, 16} : RowShape{256, 32};
}

// Two blocks per SM, fewer when the frames do not fill them.
int row_blocks(const NormArgs& a, bool bwd) {
  const int G = kRowThreads / row_shape(a.C, bwd).R;
  return std::max(1, std::min(cdiv(a.B * a.T, G), 148 * 2));
}

int time_cluster(int C) { return cdiv(C, kTimeC); }

bool aligned(const NormTensor& t, int n, int V, int elem) {
  return !t.p || (reinterpret_cast<uintptr_t>(t.p) % (V * elem) == 0 && t.b % V == 0 && t.o % V == 0 && n % V == 0);
}
bool aligned(const NormArgs& a, bool bwd, int n, int V, int elem) {
  return aligned(a.x, n, V, elem) && aligned(a.y, n, V, elem) &&
         (bwd ? aligned(a.dout, n, V, elem) && aligned(a.dx, n, V, elem) : aligned(a.out, n, V, elem));
}

// Frames per lane of the [B][C][T] kernels.
int time_vec(const NormArgs& a, bool bwd) { return aligned(a, bwd, a.T, 4, a.ty == Ty::F32 ? 4 : 2) ? 4 : 1; }

int time_per_sm(const NormArgs& a, bool bwd) {  // one block where a lane's single frames leave it many sums
  return bwd && time_vec(a, bwd) == 1 && a.C > 4 * kTimeWarps ? 1 : 2;
}
int time_teams(const NormArgs& a, int per_sm) {
  return (int)std::max<int64_t>(1, std::min<int64_t>((int64_t)a.B * cdiv(a.T, 32), 148 * per_sm / time_cluster(a.C)));
}

template <typename T, int V, int E, int R, bool BWD>
cudaError_t rows_launch(const NormArgs& a, cudaStream_t st) {
  constexpr int G = kRowThreads / R;
  const size_t stage = (size_t)G * (BWD ? 3 : 2) * a.C * sizeof(T), sums = BWD ? 2 * (size_t)a.C * sizeof(float) : 0;
  // Two blocks share an SM's shared memory where two stages of each fit.
  int stages = 0;
  if (V > 1) {
    stages = (int)std::min<size_t>(kMaxStages, 96 * 1024 / stage);
    if (stages < 2) stages = (int)(200 * 1024 / stage);
  }
  const size_t smem = std::max(stages * stage, sums);
  int regs;
  const cudaError_t e = kernel_setup(norm_rows<T, V, E, R, BWD>, smem, &regs);
  if (e != cudaSuccess) return e;
  norm_rows<T, V, E, R, BWD><<<row_blocks(a, BWD), kRowThreads, smem, st>>>(a, stages);
  return cudaGetLastError();
}

template <typename T, int V, bool BWD>
cudaError_t rows_shape(const NormArgs& a, cudaStream_t st) {
  const RowShape s = row_shape(a.C, BWD);
  if (s.R == 32 && s.E == 8) return rows_launch<T, V, 8, 32, BWD>(a, st);
  if (s.R == 32 && s.E == 16) return rows_launch<T, V, 16, 32, BWD>(a, st);
  if constexpr (BWD) {
    if (s.R == 64) return rows_launch<T, V, 16, 64, true>(a, st);
    if (s.R == 128) return rows_launch<T, V, 16, 128, true>(a, st);
    return s.E == 16 ? rows_launch<T, V, 16, 256, true>(a, st) : rows_launch<T, V, 32, 256, true>(a, st);
  } else {
    if (s.R == 32) return rows_launch<T, V, 32, 32, false>(a, st);
    if (s.R == 64) return rows_launch<T, V, 32, 64, false>(a, st);
    return s.R == 128 ? rows_launch<T, V, 32, 128, false>(a, st) : rows_launch<T, V, 32, 256, false>(a, st);
  }
}

template <typename T, int V, int E, bool BWD>
cudaError_t time_launch(const NormArgs& a, int cs, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(time_teams(a, time_per_sm(a, BWD)) * cs));
  cfg.blockDim = dim3(kTimeWarps * 32);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cs;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, norm_time<T, V, E, BWD>, a, cs);
}

// E channels of V frames per lane: as many as a block of 16 warps needs for its
// even share of C.
template <typename T, bool BWD>
cudaError_t time_shape(const NormArgs& a, cudaStream_t st) {
  const int cs = time_cluster(a.C), per = cdiv(cdiv(a.C, cs), kTimeWarps);
  if (time_vec(a, BWD) == 4) {
    if (per > 12) return time_launch<T, 4, 4, BWD>(a, cs, st);
    if (per > 8) return time_launch<T, 4, 3, BWD>(a, cs, st);
    return per > 4 ? time_launch<T, 4, 2, BWD>(a, cs, st) : time_launch<T, 4, 1, BWD>(a, cs, st);
  }
  if (per > 12) return time_launch<T, 1, 16, BWD>(a, cs, st);
  return per > 4 ? time_launch<T, 1, 12, BWD>(a, cs, st) : time_launch<T, 1, 4, BWD>(a, cs, st);
}

template <typename T, bool BWD>
cudaError_t run_t(const NormArgs& a, cudaStream_t st) {
  if (!a.rows) return time_shape<T, BWD>(a, st);
  constexpr int V = 16 / sizeof(T);
  return aligned(a, BWD, a.C, V, sizeof(T)) ? rows_shape<T, V, BWD>(a, st) : rows_shape<T, 1, BWD>(a, st);
}

template <bool BWD>
cudaError_t run(const NormArgs& a, cudaStream_t st) {
  switch (a.ty) {
    case Ty::F32: return run_t<float, BWD>(a, st);
    case Ty::F16: return run_t<__half, BWD>(a, st);
    default: return run_t<__nv_bfloat16, BWD>(a, st);
  }
}

}  // namespace

// The largest of the kernels the alignment may choose.
size_t norm_bwd_workspace(const NormArgs& a) {
  return (size_t)(a.rows ? row_blocks(a, true) : time_teams(a, 2)) * 2 * a.C * sizeof(float);
}

cudaError_t norm_forward(const NormArgs& a, cudaStream_t st) { return a.T ? run<false>(a, st) : cudaSuccess; }

cudaError_t norm_backward(const NormArgs& a, cudaStream_t st) {
  const cudaError_t e = run<true>(a, st);
  if (e != cudaSuccess) return e;
  const int n = a.rows ? row_blocks(a, true) : time_teams(a, time_per_sm(a, true));
  const PdlScope pdl(true);
  return launch_k(norm_part_sum, cdiv(2 * a.C, 32), 512, 0, st, (const float*)a.part, n, a.C, a.dgamma, a.dbeta);
}

cudaError_t norm_give_ups(int* out, cudaStream_t st) { return read_give_ups(g_give_ups, out, st); }

}  // namespace gsv
