// attn_simt.cu -- attention forward and backward for fp32 on the CUDA cores
// (formulas in attn.h).
//
// One block of 256 threads works on 64 x 64 score tiles; a thread holds 4 x 4
// scores (rows 4 ty .., columns tx + 16 c) and 4 rows x D / 16 columns of each
// accumulator (runs of 2 or 4 side by side, so that 16 threads read one run of
// a row without bank conflicts).  All operand tiles stay row-major in shared memory with a row
// pitch of D + 4 floats: a quarter warp reading float4s of consecutive rows
// then hits all 32 banks once.  Score products read 8 float4 for 64 FMAs,
// which keeps shared memory (12 wavefronts) below the FMA time (16 cycles).
// The forward walks the key tiles once with a running maximum and sum; the
// backward recomputes the probabilities from the saved log-sum-exp, once per
// key tile (dk, dv) and once per query tile (dq), so every gradient element
// is summed in a fixed order.  Products run two fp32 lanes per instruction,
// which leaves issue slots for the shared-memory reads.
//
// Where the largest tile row or column would outlast an even share of the work
// on all SMs, its tiles are dealt out to the blocks of a cluster, whose sums
// are joined in rank order through distributed shared memory.
//
// Not on the tensor cores: three 16-bit pieces per value and six products for
// each need room that a block does not have at D = 128; two TF32 pieces and
// three products have not been tried, nor their error measured.
//
// Measured on B200: backward of 4 utterances, 4 heads of 128, up to 500 queries
// and 173 keys: 87 us and 7 for the rows, 13 TFLOP/s.  The whole tiles' seven
// products would take 27 us on all SMs at the FMA rate; a block has 8 warps an
// SM (its tiles fill the shared memory) and loads the streamed tiles between
// two barriers, so that nothing covers them (FMA pipe 38 % busy, issue slots
// 32 %, 17 to 43 % from SM to SM, since the units do not divide evenly).  One
// utterance of 37 frames, 2 heads of 96, window 4, forward: 14.8 us, one tile a
// head, all of it latency.
#include <cooperative_groups.h>

#include <algorithm>

#include "attn_launch.h"
#include "attn_tc.cuh"

namespace cg = cooperative_groups;

namespace gsv {
namespace {

constexpr int kBT = 64;        // rows and columns of a score tile
constexpr int kThreads = 256;
constexpr int kLdP = kBT + 4;  // pitch of a transposed probability tile

// kBT x DP floats from global rows (nvalid of them, D channels), zeros
// elsewhere.  Addresses are clamped and values dropped afterwards, so that no
// load stands under a branch and a thread's loads are all in flight together.
template <typename T, int DP>
__device__ __forceinline__ void load_rows(float* s, const T* g, int64_t stride, int nvalid, int D, bool vec) {
  constexpr int V = DP / 4, N = kBT * V / kThreads;
  float4 o[N];
  if (nvalid > 0) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = threadIdx.x + n * kThreads, r = i / V, c = (i - r * V) * 4;
      const T* p = g + (int64_t)min(r, nvalid - 1) * stride;
      if (vec) {
        o[n] = *reinterpret_cast<const float4*>(p + min(c, D - 4));
      } else {
        o[n] = make_float4(to_f(p[min(c, D - 1)]), to_f(p[min(c + 1, D - 1)]), to_f(p[min(c + 2, D - 1)]),
                           to_f(p[min(c + 3, D - 1)]));
      }
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int i = threadIdx.x + n * kThreads, r = i / V, c = (i - r * V) * 4;
    const bool in = r < nvalid;
    float4 v;
    v.x = in && c < D ? o[n].x : 0.f;
    v.y = in && c + 1 < D ? o[n].y : 0.f;
    v.z = in && c + 2 < D ? o[n].z : 0.f;
    v.w = in && c + 3 < D ? o[n].w : 0.f;
    *reinterpret_cast<float4*>(s + r * (DP + 4) + c) = v;
  }
}

// acc[a][c] += A[4 ty + a] . B[tx + 16 c], even and odd channels apart until the end
template <int DP>
__device__ __forceinline__ void dot_tile(const float* A, const float* B, int ty, int tx, float acc[4][4]) {
  constexpr int L = DP + 4;
  F2 s[4][4] = {{F2(0.f, 0.f), F2(0.f, 0.f), F2(0.f, 0.f), F2(0.f, 0.f)},
                {F2(0.f, 0.f), F2(0.f, 0.f), F2(0.f, 0.f), F2(0.f, 0.f)},
                {F2(0.f, 0.f), F2(0.f, 0.f), F2(0.f, 0.f), F2(0.f, 0.f)},
                {F2(0.f, 0.f), F2(0.f, 0.f), F2(0.f, 0.f), F2(0.f, 0.f)}};
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
        s[a][c] = fma2(F2(x[a].x, x[a].y), F2(y[c].x, y[c].y), s[a][c]);
        s[a][c] = fma2(F2(x[a].z, x[a].w), F2(y[c].z, y[c].w), s[a][c]);
      }
  }
#pragma unroll
  for (int a = 0; a < 4; ++a)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      float lo, hi;
      s[a][c].get(lo, hi);
      acc[a][c] += lo + hi;
    }
}

// The column of a thread's accumulator w.
template <int DP>
__device__ __forceinline__ int col(int tx, int w) {
  constexpr int V = DP % 64 == 0 ? 4 : 2;
  return (w / V) * 16 * V + tx * V + w % V;
}

// acc[a][w] += sum_j P[j][4 ty + a] M[j][col(w)]
template <int DP>
__device__ __forceinline__ void acc_tile(const float* P, const float* M, int ty, int tx, float (*acc)[DP / 16]) {
  constexpr int L = DP + 4, W = DP / 16, V = DP % 64 == 0 ? 4 : 2;
#pragma unroll 4
  for (int j = 0; j < kBT; ++j) {
    const float4 p = *reinterpret_cast<const float4*>(P + j * kLdP + 4 * ty);
    const F2 pa(p.x, p.x), pb(p.y, p.y), pc(p.z, p.z), pd(p.w, p.w);
    float m[W];
#pragma unroll
    for (int w = 0; w < W; w += V) {
      const float* from = M + j * L + col<DP>(tx, w);
      if constexpr (V == 4) {
        const float4 t = *reinterpret_cast<const float4*>(from);
        m[w] = t.x, m[w + 1] = t.y, m[w + 2] = t.z, m[w + 3] = t.w;
      } else {
        const float2 t = *reinterpret_cast<const float2*>(from);
        m[w] = t.x, m[w + 1] = t.y;
      }
    }
#pragma unroll
    for (int w = 0; w < W; w += 2) {
      const F2 t(m[w], m[w + 1]);
      fma2(pa, t, F2(acc[0][w], acc[0][w + 1])).get(acc[0][w], acc[0][w + 1]);
      fma2(pb, t, F2(acc[1][w], acc[1][w + 1])).get(acc[1][w], acc[1][w + 1]);
      fma2(pc, t, F2(acc[2][w], acc[2][w + 1])).get(acc[2][w], acc[2][w + 1]);
      fma2(pd, t, F2(acc[3][w], acc[3][w + 1])).get(acc[3][w], acc[3][w + 1]);
    }
  }
}

// This thread's rows of a tile of sums, to shared memory.
template <int DP>
__device__ __forceinline__ void put_tile(float* s, int ty, int tx, float (*acc)[DP / 16]) {
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int w = 0; w < DP / 16; ++w) s[(4 * ty + x) * (DP + 4) + col<DP>(tx, w)] = acc[x][w];
}

// The cluster's sums of one tile (put_tile by every block), joined in rank order
// for the rows [from, from + 64 / cs) and handed to out(row, channel, sums of 4
// channels, weights of the ranks applied).  Each thread has all its remote reads
// of two ranks under way together; cs >= 2.
template <int DP, typename Weight, typename Out>
__device__ __forceinline__ void join_tile(cg::cluster_group& cl, int cs, int from, float* s, Weight weight, Out out) {
  constexpr int V = DP / 4, J = 64 * V / 2 / kThreads;
  const int total = kBT / cs * V;
  float4 t[J];
#pragma unroll
  for (int j = 0; j < J; ++j) t[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int x = 0; x < cs; x += 2) {
    float4 u[J], v[J];
    float wu[J], wv[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int e = min((int)threadIdx.x + j * kThreads, total - 1), y = from + e / V, d = (e % V) * 4;
      u[j] = *reinterpret_cast<const float4*>(cl.map_shared_rank(s + y * (DP + 4) + d, x));
      v[j] = *reinterpret_cast<const float4*>(cl.map_shared_rank(s + y * (DP + 4) + d, x + 1));
      wu[j] = weight(y, x);
      wv[j] = weight(y, x + 1);
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      t[j].x = fmaf(wv[j], v[j].x, fmaf(wu[j], u[j].x, t[j].x));
      t[j].y = fmaf(wv[j], v[j].y, fmaf(wu[j], u[j].y, t[j].y));
      t[j].z = fmaf(wv[j], v[j].z, fmaf(wu[j], u[j].z, t[j].z));
      t[j].w = fmaf(wv[j], v[j].w, fmaf(wu[j], u[j].w, t[j].w));
    }
  }
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int e = threadIdx.x + j * kThreads;
    if (e >= total) continue;
    const float f[4] = {t[j].x, t[j].y, t[j].z, t[j].w};
#pragma unroll
    for (int c = 0; c < 4; ++c) out(from + e / V, (e % V) * 4 + c, f[c]);
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
__global__ void __launch_bounds__(kThreads) attn_fwd_simt(const __grid_constant__ AttnArgs a, const int cs,
                                                          const bool vec) {
  constexpr int W = DP / 16;
  extern __shared__ __align__(16) float sm[];
  float* sQ = sm;
  float* sK = sQ + tile_floats<DP>();
  float* sV = sK + tile_floats<DP>();
  float* sP = sV + tile_floats<DP>();
  float* sR = sP + kBT * kLdP;  // [nrel][64]: q . relk, then the near scores
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  cg::cluster_group cl = cg::this_cluster();
  // Long rows of a causal mask first, of all heads, so that the last blocks are short ones (2 x 8 heads of 64, 1500
  // tokens: 262 -> 200 us).
  const int rank = blockIdx.x % cs, unit = blockIdx.x / cs, tile = unit / (a.H * a.B);
  const int i0 = (cdiv(a.Tq, kBT) - 1 - tile) * kBT, bh = unit - tile * a.H * a.B, b = bh / a.H, h = bh - b * a.H;
  const int ql = clamp_len(a.qlen, b, a.Tq), kl = clamp_len(a.klen, b, a.Tk), off = kl - ql;
  const int hk = h / (a.H / a.Hkv), D = a.D;
  const T* q = static_cast<const T*>(a.q) + b * a.sq.b + h * a.sq.h + (int64_t)i0 * a.sq.t;
  const T* k = static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h;
  const T* v = static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h;
  load_rows<T, DP>(sQ, q, a.sq.t, ql - i0, D, vec);
  __syncthreads();
  const T* relk = static_cast<const T*>(a.relk);
  const T* relv = static_cast<const T*>(a.relv);
  const bool rvec = vec && reinterpret_cast<uintptr_t>(relk) % 16 == 0;
  if (a.nrel) {
    load_rows<T, DP>(sV, relk, D, a.nrel, D, rvec);
    __syncthreads();
    for (int e = threadIdx.x; e < a.nrel * kBT; e += kThreads) {
      const float *x = sQ + (e % kBT) * (DP + 4), *y = sV + (e / kBT) * (DP + 4);
      float s0 = 0.f, s1 = 0.f;
#pragma unroll 8
      for (int d = 0; d < DP; d += 4) {
        const float4 u = *reinterpret_cast<const float4*>(x + d), v = *reinterpret_cast<const float4*>(y + d);
        s0 = fmaf(u.x, v.x, fmaf(u.z, v.z, s0));
        s1 = fmaf(u.y, v.y, fmaf(u.w, v.w, s1));
      }
      sR[e] = s0 + s1;
    }
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
  for (int j0 = rank * kBT; j0 < kend; j0 += cs * kBT) {
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
#pragma unroll 3
  for (int r = 0; r < a.nrel; ++r) {
    float e[W];
#pragma unroll
    for (int w = 0; w < W; ++w) e[w] = to_f(relv[r * D + min(col<DP>(tx, w), D - 1)]);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int j = i0 + 4 * ty + x + off + r - a.window;
      const float mu = m[x] == -INFINITY ? 0.f : m[x];
      const float p = j >= 0 && j < n[x] && (j / kBT & (cs - 1)) == rank ? exp2f(sR[r * kBT + 4 * ty + x] - mu) : 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) acc[x][w] = fmaf(p, e[w], acc[x][w]);
    }
  }
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int i = i0 + 4 * ty + x;
    const float mu = m[x] == -INFINITY ? 0.f : m[x];
    if (cs > 1) {
      if (tx == 0) {
        sP[4 * ty + x] = m[x];
        sP[kBT + 4 * ty + x] = l[x];
      }
      continue;
    }
    if (i >= a.Tq) continue;
    const float inv = l[x] == 0.f ? 0.f : 1.f / l[x];
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (col<DP>(tx, w) < D) o[(int64_t)i * a.so.t + col<DP>(tx, w)] = from_f<T>(l[x] == 0.f ? 0.f : acc[x][w] * inv);
    if (tx == 0 && a.lse)
      a.lse[((int64_t)b * a.H + h) * a.Tq + i] = l[x] == 0.f ? -INFINITY : (mu + log2f(l[x])) * kLn2;
  }
  if (cs == 1) return;
  put_tile<DP>(sQ, ty, tx, acc);
  cl.sync();
  // The ranks' weights of each row that this block writes, and the row's sum.
  const int per = kBT / cs, from = rank * per;
  float* sw = sK;             // [row][rank]
  float* sl = sK + kBT * 8;   // [row]
  if ((int)threadIdx.x < per) {
    const int y = from + threadIdx.x;
    float M = -INFINITY, L = 0.f;
    for (int x = 0; x < cs; ++x) M = fmaxf(M, *cl.map_shared_rank(sP + y, x));
    for (int x = 0; x < cs; ++x) {
      const float mx = *cl.map_shared_rank(sP + y, x), f = mx == -INFINITY ? 0.f : exp2f(mx - M);
      sw[y * 8 + x] = f;
      L = fmaf(f, *cl.map_shared_rank(sP + kBT + y, x), L);
    }
    sl[y] = L;
    if (i0 + y < a.Tq && a.lse)
      a.lse[((int64_t)b * a.H + h) * a.Tq + i0 + y] =
          L == 0.f ? -INFINITY : ((M == -INFINITY ? 0.f : M) + log2f(L)) * kLn2;
  }
  __syncthreads();
  join_tile<DP>(
      cl, cs, from, sQ, [&](int y, int x) { return sw[y * 8 + x]; },
      [&](int y, int d, float t) {
        if (i0 + y < a.Tq && d < D)
          o[(int64_t)(i0 + y) * a.so.t + d] = from_f<T>(sl[y] == 0.f ? 0.f : t / sl[y]);
      });
  cl.sync();  // the block's sums have been read
}

// The first units (clusters) take dk, dv of one key tile and key head each, the
// others dq of one query tile and head: the keys' units, which take a third
// longer a tile, all start before the queries'.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) attn_bwd_simt(const __grid_constant__ AttnArgs a,
                                                          const __grid_constant__ BwdWs ws, const int nk, const int cs,
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
  const int D = a.D, g = a.H / a.Hkv, nq = cdiv(a.Tq, kBT);
  const int rank = blockIdx.x % cs, unit = blockIdx.x / cs, kunits = nk * a.Hkv * a.B;
  const bool keys = unit < kunits;
  // Tiles slowest, the longest ones of a causal call first.
  const int heads = (keys ? a.Hkv : a.H) * a.B, at = keys ? unit : unit - kunits;
  const int tile = keys ? at / heads : nq - 1 - at / heads, bhu = at % heads;
  const int b = keys ? bhu / a.Hkv : bhu / a.H;
  const int ql = clamp_len(a.qlen, b, a.Tq), kl = clamp_len(a.klen, b, a.Tk), off = kl - ql;
  const float sl2 = a.scale * kLog2e;
  cg::cluster_group cl = cg::this_cluster();
  const int from = rank * (kBT / cs);  // first of the rows that this block writes
  auto one = [](int, int) { return 1.f; };
  if (keys) {
    const int hk = bhu - b * a.Hkv, j0 = tile * kBT;
    load_rows<T, DP>(s0, static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h + (int64_t)j0 * a.sk.t, a.sk.t,
                     kl - j0, D, vec);
    load_rows<T, DP>(s1, static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h + (int64_t)j0 * a.sv.t, a.sv.t,
                     kl - j0, D, vec);
    float dk[4][W] = {}, dv[4][W] = {};
    // From the first query that sees the tile: those without a key (they may hold anything) stay out of its sums.
    const int first = j0 >= kl ? ql : (a.causal ? max(0, j0 - off) : 0);
    for (int hh = 0; hh < g; ++hh) {
      const int h = hk * g + hh;
      const int64_t bh = (int64_t)b * a.H + h;
      for (int i0 = first + rank * kBT; i0 < ql; i0 += cs * kBT) {
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
    if (cs > 1) {
      __syncthreads();
      put_tile<DP>(s0, ty, tx, dk);
      put_tile<DP>(s1, ty, tx, dv);
      cl.sync();
      join_tile<DP>(cl, cs, from, s0, one, [&](int y, int d, float t) {
        if (j0 + y < a.Tk && d < D) odk[(int64_t)(j0 + y) * a.sdk.t + d] = from_f<T>(t * a.scale);
      });
      join_tile<DP>(cl, cs, from, s1, one, [&](int y, int d, float t) {
        if (j0 + y < a.Tk && d < D) odv[(int64_t)(j0 + y) * a.sdv.t + d] = from_f<T>(t);
      });
      cl.sync();
      return;
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int j = j0 + 4 * ty + x;
      if (j >= a.Tk) continue;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int d = col<DP>(tx, w);
        if (d >= D) continue;
        odk[(int64_t)j * a.sdk.t + d] = from_f<T>(dk[x][w] * a.scale);
        odv[(int64_t)j * a.sdv.t + d] = from_f<T>(dv[x][w]);
      }
    }
    return;
  }
  const int h = bhu - b * a.H, hk = h / g, i0 = tile * kBT;
  const int64_t bh = bhu, row = bh * a.Tq;
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
  for (int j0 = rank * kBT; j0 < kend; j0 += cs * kBT) {
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
#pragma unroll 3
  for (int r = 0; r < a.nrel; ++r) {
    float e[W];
#pragma unroll
    for (int w = 0; w < W; ++w) e[w] = to_f(relk[r * D + min(col<DP>(tx, w), D - 1)]);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = i0 + 4 * ty + x, j = i + off + r - a.window;
      const bool use = j >= 0 && j < n[x] && (j / kBT & (cs - 1)) == rank;
      const float ds = use ? ws.sband[(row + i) * a.nrel + r] : 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) dq[x][w] = fmaf(ds, e[w], dq[x][w]);
    }
  }
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int i = i0 + 4 * ty + x;
    if (cs > 1 || i >= a.Tq) continue;
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (col<DP>(tx, w) < D) o[(int64_t)i * a.sdq.t + col<DP>(tx, w)] = from_f<T>(dq[x][w] * a.scale);
  }
  if (cs == 1) return;
  put_tile<DP>(s0, ty, tx, dq);
  cl.sync();
  join_tile<DP>(cl, cs, from, s0, one, [&](int y, int d, float t) {
    if (i0 + y < a.Tq && d < D) o[(int64_t)(i0 + y) * a.sdq.t + d] = from_f<T>(t * a.scale);
  });
  cl.sync();
}

// Blocks per tile row or column (a unit): the power of two with the smallest
// estimate of the time, the longer of the longest unit's share and an even
// share of all work on the SMs, where each block adds `set_up` (resident tiles,
// joining).  One utterance of 500, 2 heads of 96, window 4: 65 -> 36 us forward;
// backward 126 -> 53, and 79 with twice as many.  The cross case above: 143 ->
// 94, and 129 with twice as many.
int split(int64_t longest, int64_t total, int64_t units, int set_up, int tiles) {
  int best = 1;
  int64_t least = INT64_MAX;
  for (int cs = 1; cs <= 8 && cs <= tiles; cs *= 2) {
    const int64_t t = std::max(((longest + cs - 1) / cs + set_up) * 148, total + units * cs * set_up);
    if (t < least) {
      least = t;
      best = cs;
    }
  }
  return best;
}

template <typename... K, typename... A>
cudaError_t launch_split(void (*kern)(K...), dim3 grid, int cs, size_t smem, cudaStream_t st, A... args) {
  int regs;
  const cudaError_t e = kernel_setup(kern, smem, &regs);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cs;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

template <typename T, int DP>
cudaError_t fwd(const AttnArgs& a, cudaStream_t st) {
  const size_t smem = sizeof(float) * (3 * tile_floats<DP>() + kBT * kLdP + a.nrel * kBT);
  const int el = sizeof(T);
  const bool vec = attn_rows_aligned(a.q, a.sq, a.D, el) && attn_rows_aligned(a.k, a.sk, a.D, el) &&
                   attn_rows_aligned(a.v, a.sv, a.D, el);
  const int nq = cdiv(a.Tq, kBT), nk = cdiv(a.Tk, kBT);
  const int64_t units = (int64_t)a.B * a.H * nq;
  const int cs = split(nk, units * nk, units, 2, nk);  // in tiles
  return launch_split(attn_fwd_simt<T, DP>, dim3((unsigned)(units * cs)), cs, smem, st, a, cs, vec);
}

template <typename T, int DP>
cudaError_t bwd(const AttnArgs& a, const BwdWs& ws, cudaStream_t st) {
  const size_t smem = sizeof(float) * (4 * tile_floats<DP>() + 2 * kBT * kLdP);
  const int el = sizeof(T);
  const bool vec = attn_rows_aligned(a.q, a.sq, a.D, el) && attn_rows_aligned(a.k, a.sk, a.D, el) &&
                   attn_rows_aligned(a.v, a.sv, a.D, el) && attn_rows_aligned(a.dout, a.sdo, a.D, el);
  const int nk = cdiv(a.Tk, kBT), nq = cdiv(a.Tq, kBT);
  // In products: four a tile for the keys' gradients, three for the queries'.
  const int g = a.H / a.Hkv;
  const int64_t units = ((int64_t)nk * a.Hkv + (int64_t)nq * a.H) * a.B;
  const int cs = split(std::max(4 * (int64_t)g * nq, 3 * (int64_t)nk), (int64_t)7 * a.B * a.H * nq * nk, units, 4,
                       std::max(nq, nk));
  return launch_split(attn_bwd_simt<T, DP>, dim3((unsigned)(units * cs)), cs, smem, st, a, ws, nk, cs, vec);
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
