// attn_rows.cu -- the attention backward's per-row pass and the gradients of
// the relative keys and values, and the choice of kernels of both directions.
#include <algorithm>

#include "attn_launch.h"
#include "attn_tc.cuh"
#include "gsv_pdl.cuh"

namespace gsv {
namespace {

constexpr int kFewKeys = 32;

template <int G>
__device__ __forceinline__ float group_sum(float v) {  // over aligned groups of G lanes
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ float dot8(const float* a, const float* b) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = fmaf(a[i], b[i], s);
  return s;
}

// G lanes share one row, 8 channels each; a group takes U rows, whose loads are
// all under way together.  The products with the relative rows are taken from
// shared memory by one thread per row and three offsets (a fifth of the
// instructions of products shared by G lanes, most of which were reductions).
// Query rows: delta = do . o in fp32
// and the products with the relative rows; fp16 adds the norms of the rows of
// do and v.
//
// The o given here carries its rounding to 16 bits and that of the forward's
// probabilities, which reach ds through delta as p_ij |do| |o's error|.  Where
// the probabilities spread over many keys o shrinks against v and the term
// disappears; where a row rests on one key it stays, about as large as the
// rounding of that ds.  Rows of up to kFewKeys keys, where that is the rule, take
// delta = sum_j p_ij dp_ij instead (fp32 inputs have no such rounding).
//
// Reads do and o (with a window q) once: 2 x 16 heads of 64, 4096 causal rows,
// bf16, 25 us, where the 32 rows of few keys of each head take longest; 16
// utterances of up to 500 rows, 2 heads of 96, window 4, 12 us, one or two
// blocks an SM that wait for memory twice and then do 18 products a row.
template <typename T, int G, int U>
__global__ void __launch_bounds__(kRowThreads, 4) bwd_rows_kernel(const __grid_constant__ AttnArgs a,
                                                                  const __grid_constant__ BwdWs ws,
                                                                  const int qblocks, const bool vec) {
  extern __shared__ __align__(16) float sm[];  // relk, relv as [nrel][P], then q, do as [R U][P]
  constexpr bool F16 = std::is_same<T, __half>::value, kExact = std::is_same<T, float>::value;
  constexpr int L = 8 * G, P = L + 4, R = kRowThreads / G;
  // Heads fastest: the blocks of the first rows, which take longest (few keys), start first.
  const bool key_rows = F16 && (int)blockIdx.x >= qblocks;
  const int unit = blockIdx.x - (key_rows ? qblocks : 0), hn = key_rows ? a.Hkv : a.H;
  const int tile = unit / (hn * a.B), bh32 = unit - tile * (hn * a.B);
  const int D = a.D, lane = threadIdx.x % G, d0 = lane * 8, b = bh32 / hn, h = bh32 - b * hn;
  const int ql = clamp_len(a.qlen, b, a.Tq), kl = clamp_len(a.klen, b, a.Tk);
  // Rows of the block: i0 + u R + group.
  const int i0 = tile * R * U + threadIdx.x / G;
  Raw8<T> rg[U], ro[U], rq[U];
  if (!key_rows) {
    const T* g = static_cast<const T*>(a.dout) + b * a.sdo.b + h * a.sdo.h;
    const T* o = static_cast<const T*>(a.o) + b * a.so.b + h * a.so.h;
    const T* q = static_cast<const T*>(a.q) + b * a.sq.b + h * a.sq.h;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + u * R, a.Tq - 1);  // its values are dropped where the row has no keys
      rg[u].load(g + i * a.sdo.t, d0, D, vec);
      ro[u].load(o + i * a.so.t, d0, D, vec);
      if (a.nrel) rq[u].load(q + i * a.sq.t, d0, D, vec);
    }
  } else {
    const T* v = static_cast<const T*>(a.v) + b * a.sv.b + h * a.sv.h;
#pragma unroll
    for (int u = 0; u < U; ++u) rg[u].load(v + min(i0 + u * R, a.Tk - 1) * a.sv.t, d0, D, vec);
  }
  float* srk = sm;
  float* srv = srk + a.nrel * P;
  float* srows = srv + a.nrel * P;  // q; do R U P later
  for (int e = threadIdx.x; e < a.nrel * L; e += kRowThreads) {
    const int r = e / L, d = e % L;
    const T k = static_cast<const T*>(a.relk)[r * D + min(d, D - 1)], v = static_cast<const T*>(a.relv)[r * D + min(d, D - 1)];
    srk[r * P + d] = d < D ? to_f(k) : 0.f;
    srv[r * P + d] = d < D ? to_f(v) : 0.f;
  }
  if (a.nrel && !key_rows) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float q[8], g[8];
      rq[u].get(q);
      rg[u].get(g);
      float4* to = reinterpret_cast<float4*>(srows + (u * R + threadIdx.x / G) * P + d0);
      to[0] = make_float4(q[0], q[1], q[2], q[3]);
      to[1] = make_float4(q[4], q[5], q[6], q[7]);
      to += R * U * P / 4;
      to[0] = make_float4(g[0], g[1], g[2], g[3]);
      to[1] = make_float4(g[4], g[5], g[6], g[7]);
    }
  }
  if (a.nrel) __syncthreads();
  if (key_rows) {
    float ev = 0.f;  // largest |relv|^2
    if ((threadIdx.x & 31) < a.nrel)
      for (int d = 0; d < L; ++d) ev = fmaf(srv[(threadIdx.x & 31) * P + d], srv[(threadIdx.x & 31) * P + d], ev);
    ev = sqrtf(warp_max(ev));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = i0 + u * R;
      float v[8];
      rg[u].get(v);
      const float s = group_sum<G>(dot8(v, v));
      if (j < kl && lane == 0) ws.nv[((int64_t)b * a.Hkv + h) * a.Tk + j] = sqrtf(s) + ev;
    }
    return;
  }
  const float sl2 = a.scale * kLog2e;
  const int64_t bh = (int64_t)b * a.H + h;
  float delta[U], lse2[U], norm[U];
  int n[U];
  bool any_few = false;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = i0 + u * R;
    n[u] = i < a.Tq ? allowed_keys(i, ql, kl, a.causal) : 0;
    lse2[u] = a.lse[bh * a.Tq + min(i, a.Tq - 1)] * kLog2e;
    any_few = any_few || (n[u] > 0 && n[u] <= kFewKeys);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float g[8], o[8];
    rg[u].get(g);
    ro[u].get(o);
    delta[u] = group_sum<G>(dot8(g, o));
    norm[u] = F16 ? sqrtf(group_sum<G>(dot8(g, g))) : 0.f;
    if (n[u] == 0) delta[u] = norm[u] = 0.f, lse2[u] = INFINITY;
  }
  if (a.nrel) {
    const int base = tile * R * U;
    constexpr int O = 3;  // offsets per thread: q and do are read once for three
    const int groups = (a.nrel + O - 1) / O;
    for (int e = threadIdx.x; e < groups * R * U; e += kRowThreads) {
      const int y = e % (R * U), r0 = e / (R * U) * O, i = base + y;
      const float4* q = reinterpret_cast<const float4*>(srows + y * P);
      const float4* g = q + R * U * P / 4;
      const float4 *rk[O], *rv[O];
      F2 x[O], z[O];
#pragma unroll
      for (int o = 0; o < O; ++o) {
        rk[o] = reinterpret_cast<const float4*>(srk + min(r0 + o, a.nrel - 1) * P);
        rv[o] = reinterpret_cast<const float4*>(srv + min(r0 + o, a.nrel - 1) * P);
        x[o] = z[o] = F2(0.f, 0.f);
      }
#pragma unroll 2
      for (int c = 0; c < L / 4; ++c) {
        const float4 a4 = q[c], c4 = g[c];
#pragma unroll
        for (int o = 0; o < O; ++o) {
          const float4 b4 = rk[o][c], d4 = rv[o][c];
          x[o] = fma2(F2(a4.x, a4.y), F2(b4.x, b4.y), x[o]);
          x[o] = fma2(F2(a4.z, a4.w), F2(b4.z, b4.w), x[o]);
          z[o] = fma2(F2(c4.x, c4.y), F2(d4.x, d4.y), z[o]);
          z[o] = fma2(F2(c4.z, c4.w), F2(d4.z, d4.w), z[o]);
        }
      }
      if (i >= ws.blocks * kRowBlock) continue;
      const bool in = i < a.Tq && allowed_keys(i, ql, kl, a.causal) > 0;
      float* rel = rel_at(ws, bh, i, a.nrel);
#pragma unroll
      for (int o = 0; o < O; ++o) {
        if (r0 + o >= a.nrel) continue;
        float lo, hi;
        x[o].get(lo, hi);
        rel[r0 + o] = in ? lo + hi : 0.f;
        z[o].get(lo, hi);
        rel[kRowBlock * a.nrel + r0 + o] = in ? lo + hi : 0.f;
      }
    }
  }
  if (!kExact && __any_sync(0xffffffffu, any_few)) {
    // The warp takes its rows in turn, one key per lane; q and do come again, broadcast to the warp.
    const int hk = h / (a.H / a.Hkv), wl = threadIdx.x & 31;
    const T* k = static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h;
    const T* v = static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h;
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll 1
      for (int from = 0; from < 32; from += G) {
        const int nr = __shfl_sync(0xffffffffu, n[u], from);
        if (nr == 0 || nr > kFewKeys) continue;
        const int ir = __shfl_sync(0xffffffffu, i0 + u * R, from), j = min(wl, nr - 1);
        const float lr = __shfl_sync(0xffffffffu, lse2[u], from);
        const T* q = static_cast<const T*>(a.q) + b * a.sq.b + h * a.sq.h + ir * a.sq.t;
        const T* g = static_cast<const T*>(a.dout) + b * a.sdo.b + h * a.sdo.h + ir * a.sdo.t;
        const unsigned r = (unsigned)(j - (ir + kl - ql) + a.window);
        const bool near = r < (unsigned)a.nrel;
        float sc = 0.f, dp = 0.f;
#pragma unroll 4
        for (int c = 0; c < D; c += 8) {
          Raw8<T> kr, vr, qr, gr;
          kr.load(k + j * a.sk.t, c, D, vec);
          vr.load(v + j * a.sv.t, c, D, vec);
          qr.load(q, c, D, vec);
          gr.load(g, c, D, vec);
          float kk[8], vv[8], qq[8], gg[8];
          kr.get(kk);
          vr.get(vv);
          qr.get(qq);
          gr.get(gg);
          if (near)
#pragma unroll
            for (int y = 0; y < 8; ++y) kk[y] += srk[r * P + c + y], vv[y] += srv[r * P + c + y];
          sc += dot8(qq, kk);
          dp += dot8(gg, vv);
        }
        const float t = group_sum<32>(wl < nr ? exp2f(fmaf(sc, sl2, -lr)) * dp : 0.f);
        if (threadIdx.x % 32 / G == from / G) delta[u] = t;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = i0 + u * R;
    if (lane != 0 || i >= ws.blocks * kRowBlock) continue;
    float* rw = row_at(ws, bh, i);
    rw[0] = (F16 ? kHalfShift : 0.f) - lse2[u];
    rw[kRowBlock] = -delta[u];
    if (F16 && i < a.Tq) ws.ndo[bh * a.Tq + i] = norm[u];
  }
}

// fp32: partial sums over kRelRows query rows of one head: thread (d, half)
// holds channel d of every offset over one half of the rows.  Fixed row order, so
// the result does not depend on scheduling.
template <int NR>
__global__ void __launch_bounds__(2 * kAttnMaxD) bwd_rel_kernel(const AttnArgs a, const BwdWs ws) {
  __shared__ float sp[kRelRows][NR], ss[kRelRows][NR];
  __shared__ float red[2 * NR][kAttnMaxD];
  const int tiles = cdiv(a.Tq, kRelRows), bh = blockIdx.x / tiles, i0 = (blockIdx.x - bh * tiles) * kRelRows;
  const int b = bh / a.H, h = bh - b * a.H, D = a.D;
  const int ql = clamp_len(a.qlen, b, a.Tq), kl = clamp_len(a.klen, b, a.Tk);
  for (int e = threadIdx.x; e < kRelRows * NR; e += 2 * kAttnMaxD) {
    const int y = e / NR, r = e - y * NR, i = i0 + y, j = i + kl - ql - a.window + r;
    const bool in = r < a.nrel && j >= 0 && j < allowed_keys(i, ql, kl, a.causal);
    const int64_t at = ((int64_t)bh * a.Tq + i) * a.nrel + r;
    ss[y][r] = in ? ws.sband[at] : 0.f;
    sp[y][r] = in ? ws.pband[at] : 0.f;
  }
  __syncthreads();
  const int d = threadIdx.x % kAttnMaxD, half = threadIdx.x / kAttnMaxD;
  float ak[NR] = {}, av[NR] = {};
  const float* q = static_cast<const float*>(a.q) + b * a.sq.b + h * a.sq.h + d;
  const float* g = static_cast<const float*>(a.dout) + b * a.sdo.b + h * a.sdo.h + d;
  const int y0 = max(half * (kRelRows / 2), first_query(ql, kl, a.causal) - i0);
  const int y1 = min(half * (kRelRows / 2) + kRelRows / 2, ql - i0);
#pragma unroll 4
  for (int y = y0; y < y1; ++y) {
    const float qv = d < D ? q[(int64_t)(i0 + y) * a.sq.t] : 0.f;
    const float gv = d < D ? g[(int64_t)(i0 + y) * a.sdo.t] : 0.f;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      ak[r] = fmaf(ss[y][r], qv, ak[r]);
      av[r] = fmaf(sp[y][r], gv, av[r]);
    }
  }
  if (half == 1)
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      red[r][d] = ak[r];
      red[NR + r][d] = av[r];
    }
  __syncthreads();
  if (half == 1 || d >= D) return;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    if (r >= a.nrel) continue;
    ws.part[((int64_t)blockIdx.x * 2 * a.nrel + r) * D + d] = (ak[r] + red[r][d]) * a.scale;
    ws.part[((int64_t)blockIdx.x * 2 * a.nrel + a.nrel + r) * D + d] = av[r] + red[NR + r][d];
  }
}

// 32 sums per block, its 16 warps taking every 16th partial sum.
template <typename T>
__global__ void __launch_bounds__(512) bwd_rel_sum_kernel(const AttnArgs a, const BwdWs ws, const int64_t blocks) {
  __shared__ float s[16][32];
  pdl_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int n = a.nrel * a.D, e = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (e < 2 * n) {
#pragma unroll 4
    for (int64_t x = w; x < blocks; x += 16) v += ws.part[x * 2 * n + e];
  }
  s[w][lane] = v;
  __syncthreads();
  if (w != 0 || e >= 2 * n) return;
  for (int x = 1; x < 16; ++x) v += s[x][lane];
  if (e < n) static_cast<T*>(a.drelk)[e] = from_f<T>(v);
  else static_cast<T*>(a.drelv)[e - n] = from_f<T>(v);
}

template <typename T, int G>
cudaError_t rows_g(const AttnArgs& a, const BwdWs& ws, cudaStream_t st) {
  constexpr int U = kRowTurns, R = kRowThreads / G * U;
  const RowBlocks n = row_blocks(a);
  const size_t smem = a.nrel ? sizeof(float) * 2 * (a.nrel + R) * (8 * G + 4) : 0;
  int regs;
  const cudaError_t e = kernel_setup(bwd_rows_kernel<T, G, U>, smem, &regs);
  if (e != cudaSuccess) return e;
  const int el = sizeof(T);
  const bool vec = attn_rows_aligned(a.q, a.sq, a.D, el) && attn_rows_aligned(a.o, a.so, a.D, el) &&
                   attn_rows_aligned(a.dout, a.sdo, a.D, el) && attn_rows_aligned(a.k, a.sk, a.D, el) &&
                   attn_rows_aligned(a.v, a.sv, a.D, el) && a.D % 8 == 0;
  bwd_rows_kernel<T, G, U><<<(unsigned)(n.q + n.k), kRowThreads, smem, st>>>(a, ws, (int)n.q, vec);
  return cudaGetLastError();
}

template <typename T>
cudaError_t rows_t(const AttnArgs& a, const BwdWs& ws, cudaStream_t st) {
  const int g = row_lanes(a.D);
  return g == 4 ? rows_g<T, 4>(a, ws, st) : g == 8 ? rows_g<T, 8>(a, ws, st) : rows_g<T, 16>(a, ws, st);
}

template <typename T>
cudaError_t rel_t(const AttnArgs& a, const BwdWs& ws, cudaStream_t st) {
  const int64_t blocks = rel_blocks(a);
  if (std::is_same<T, float>::value && blocks > 0) {
    if (a.nrel <= 9) bwd_rel_kernel<9><<<(unsigned)blocks, 2 * kAttnMaxD, 0, st>>>(a, ws);
    else bwd_rel_kernel<2 * kAttnMaxWindow + 1><<<(unsigned)blocks, 2 * kAttnMaxD, 0, st>>>(a, ws);
  }
  const PdlScope pdl(blocks > 0);
  return launch_k(bwd_rel_sum_kernel<T>, cdiv(2 * a.nrel * a.D, 32), 512, 0, st, a, ws, blocks);
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
  // A tile kernel would fill 64 or 128 rows for these: 28 us (fp16) and 144 us (fp32) against 12 for one token of
  // 16 sequences, 16 heads of 32 over 4 key heads and up to 1531 keys.
  if ((int64_t)a.Tq * (a.H / a.Hkv) <= kFewRows) return attn_fwd_few_rows(a, st);
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
