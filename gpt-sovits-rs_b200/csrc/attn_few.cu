// attn_few.cu -- attention forward for few queries per key head (a decoding
// step), all types, fp32 arithmetic (formulas in attn.h).
//
// With at most kFewRows rows (queries times query heads per key head) the call
// is bound by reading k and v once.  Each row of k and v is read by G lanes, 8
// channels each, as 16-byte vectors, and serves all rows of its key head from
// registers.  Every group of G lanes walks its own keys, 64 bytes of k and of v
// per lane at a time, with its own running maximum and sum, so nothing is
// exchanged until the end; then groups, warps and the blocks of a cluster
// (which split the keys) are joined in a fixed order, the last through
// distributed shared memory: one launch and no workspace.
//
// A lane copies its own pieces to shared memory kFewStages - 1 steps ahead and
// reads them back itself, so no barrier stands in the loop (loading to registers
// instead: 68 against 47 us below).  Code that runs once per launch comes from
// memory: the relative terms are a table of products with q, filled ahead of
// the keys, and a table of near scores, used after them, instead of branches
// in the unrolled products (18.5 -> 10.2 us for 8 heads over 300 keys).
//
// Measured: 16 sequences, 8 heads of 128, 4096 keys, bf16: 47 us, 5.7 TB/s (87 %
// of a copy's bandwidth).  16 heads of 32 over 4 key heads, 16 sequences of up
// to 1531 keys, fp16: 12.3 us against 1.4 us of traffic; three dependent trips
// to memory (lengths, rows, join), the launch and two steps of arithmetic.
#include <cooperative_groups.h>

#include <algorithm>

#include "attn_launch.h"
#include "attn_tc.cuh"

namespace cg = cooperative_groups;

namespace gsv {
namespace {

constexpr int kFewWarps = 8;
constexpr int kFewSplits = 16;  // largest cluster
constexpr int kFewStages = 3;   // steps under way per lane

// With two pieces per lane (P = 2) a warp's copy takes every other 16 bytes of a
// row: through L1, so that the second one finds its sectors there.
template <int P>
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {
  if constexpr (P == 1) cp_async16(dst, src, on ? 16 : 0);
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint4 read16(uint32_t at) {
  uint4 u;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(at) : "memory");
  return u;
}

// exp2(x - m) with -inf - -inf = -inf.
__device__ __forceinline__ float ex2_from(float x, float m) { return x == -INFINITY ? 0.f : exp2f(x - m); }

template <typename T, int G, int R>
__global__ void __launch_bounds__(kFewWarps * 32, R == 8 ? 1 : 2) attn_fwd_few(const __grid_constant__ AttnArgs a, const int cs,
                                                               const bool vec) {
  constexpr int KG = 32 / G, U = sizeof(T) == 4 ? 2 : 4, DP = 8 * G;  // key groups per warp, keys per step
  constexpr int P = sizeof(T) / 2;  // 16-byte pieces of a lane's channels
  extern __shared__ __align__(16) uint4 s_ring[];  // [stage][k, v][U][P][thread]: each lane reads back its own
  __shared__ float s_acc[kFewWarps][R][DP];
  __shared__ float s_m[kFewWarps][R], s_l[kFewWarps][R];
  __shared__ float b_acc[R][DP], b_m[R], b_l[R];  // the block's, read by the cluster
  __shared__ float s_rel[R][2 * kAttnMaxWindow + 1], s_near[R][2 * kAttnMaxWindow + 1];  // q relk^T; near scores seen
  cg::cluster_group cl = cg::this_cluster();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, gl = lane % G, d0 = gl * 8;
  const int rank = blockIdx.x % cs, hk = blockIdx.y, b = blockIdx.z, D = a.D, g = a.H / a.Hkv;
  const int ql = clamp_len(a.qlen, b, a.Tq), kl = clamp_len(a.klen, b, a.Tk), off = kl - ql;
  const int rows = a.Tq * g;
  const float sl2 = a.scale * kLog2e;
  const T* relk = static_cast<const T*>(a.relk);
  const T* relv = static_cast<const T*>(a.relv);
  int n[R], ipos[R], most = 0;  // ipos: the key of the first offset
#pragma unroll
  for (int r = 0; r < R; ++r) {
    n[r] = r < rows ? allowed_keys(r / g, ql, kl, a.causal) : 0;
    ipos[r] = r / g + off - a.window;
    most = max(most, n[r]);
  }
  const T* k = static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h;
  const T* v = static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h;
  // The cluster's groups take runs of U keys in turn.
  const int groups = cs * kFewWarps * KG, mine = (rank * kFewWarps + w) * KG + lane / G;
  const int steps = (most + U * groups - 1) / (U * groups);  // the same for the whole cluster
  const uint32_t slot = (uint32_t)__cvta_generic_to_shared(s_ring) + threadIdx.x * 16;
  constexpr uint32_t kPiece = kFewWarps * 32 * 16, kOf = U * P * kPiece;
  auto fetch = [&](int x) {
    if (x < steps) {
      const int j0 = (x * groups + mine) * U;
      const uint32_t to = slot + x % kFewStages * (2 * kOf);
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t j = min(j0 + u, most - 1);
          const T* row = z ? v + j * a.sv.t : k + j * a.sk.t;
          const uint32_t at = to + z * kOf + u * P * kPiece;
          if (vec) {
#pragma unroll
            for (int y = 0; y < P; ++y)
              copy16<P>(at + y * kPiece, reinterpret_cast<const uint4*>(row + min(d0, D - 8)) + y, d0 < D);
          } else {
            Raw8<T> raw;
            raw.load(row, d0, D, false);
#pragma unroll
            for (int y = 0; y < P; ++y)
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + y * kPiece), "r"(raw.u[y].x),
                           "r"(raw.u[y].y), "r"(raw.u[y].z), "r"(raw.u[y].w)
                           : "memory");
          }
        }
    }
    cp_commit();
  };
#pragma unroll
  for (int x = 0; x < kFewStages - 1; ++x) fetch(x);
  float q[R][8], acc[R][8] = {}, m[R], l[R] = {};
  {  // all rows' loads under way together
    Raw8<T> x[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int y = min(r, rows - 1), i = y / g, h = hk * g + y - i * g;
      x[r].load(static_cast<const T*>(a.q) + b * a.sq.b + h * a.sq.h + i * a.sq.t, d0, D, vec);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m[r] = -INFINITY;
      x[r].get(q[r]);
#pragma unroll
      for (int y = 0; y < 8; ++y) q[r][y] = n[r] > 0 ? q[r][y] : 0.f;
    }
  }
  if (a.nrel) {  // the same for the whole call
    for (int e = threadIdx.x; e < R * a.nrel; e += kFewWarps * 32) s_near[e % R][e / R] = -INFINITY;
    for (int o0 = 0; o0 < a.nrel; o0 += kFewWarps * KG) {
      const int o = o0 + w * KG + lane / G;
      float e[8];
#pragma unroll
      for (int y = 0; y < 8; ++y) e[y] = d0 + y < D ? to_f(relk[min(o, a.nrel - 1) * D + d0 + y]) : 0.f;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float t = 0.f;
#pragma unroll
        for (int y = 0; y < 8; ++y) t = fmaf(q[r][y], e[y], t);
#pragma unroll
        for (int z = G / 2; z > 0; z >>= 1) t += __shfl_xor_sync(0xffffffffu, t, z);
        if (gl == 0 && o < a.nrel) s_rel[r][o] = t;
      }
    }
    __syncthreads();
  }
  for (int x = 0; x < steps; ++x) {
    const int j0 = (x * groups + mine) * U;
    fetch(x + kFewStages - 1);
    cp_wait<kFewStages - 1>();
    const uint32_t from = slot + x % kFewStages * (2 * kOf);
    auto piece = [&](int z, int u, float* f) {
      Raw8<T> raw;
#pragma unroll
      for (int y = 0; y < P; ++y) raw.u[y] = read16(from + z * kOf + (u * P + y) * kPiece);
      raw.get(f);
    };
    float s[R][U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float kk[8];
      piece(0, u, kk);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        s[r][u] = 0.f;
#pragma unroll
        for (int y = 0; y < 8; ++y) s[r][u] = fmaf(q[r][y], kk[y], s[r][u]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float mx = m[r], sum = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) s[r][u] += __shfl_xor_sync(0xffffffffu, s[r][u], o);
        const unsigned o = (unsigned)(j0 + u - ipos[r]);
        const bool near = o < (unsigned)a.nrel && j0 + u < n[r];
        if (near) s[r][u] += s_rel[r][o];
        s[r][u] = j0 + u < n[r] ? s[r][u] * sl2 : -INFINITY;
        if (near && gl == 0) s_near[r][o] = s[r][u];
        mx = fmaxf(mx, s[r][u]);
      }
      const float alpha = ex2_from(m[r], mx);
      m[r] = mx;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[r][u] = ex2_from(s[r][u], mx);
        sum += s[r][u];
      }
      l[r] = fmaf(l[r], alpha, sum);
#pragma unroll
      for (int y = 0; y < 8; ++y) acc[r][y] *= alpha;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float vv[8];
      piece(1, u, vv);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        // The last key of a run that ends early is read twice, with p = 0.
#pragma unroll
        for (int y = 0; y < 8; ++y) acc[r][y] = fmaf(s[r][u], vv[y], acc[r][y]);
      }
    }
  }
  // Groups of the warp, then its sums to shared memory.
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float M = m[r];
#pragma unroll
    for (int o = G; o < 32; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float f = ex2_from(m[r], M);
    l[r] *= f;
#pragma unroll
    for (int o = G; o < 32; o <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
#pragma unroll
    for (int y = 0; y < 8; ++y) {
      acc[r][y] *= f;
#pragma unroll
      for (int o = G; o < 32; o <<= 1) acc[r][y] += __shfl_xor_sync(0xffffffffu, acc[r][y], o);
      if (lane < G) s_acc[w][r][d0 + y] = acc[r][y];
    }
    if (lane == 0) {
      s_m[w][r] = M;
      s_l[w][r] = l[r];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < R * DP; e += kFewWarps * 32) {
    const int r = e / DP, d = e - r * DP;
    float M = -INFINITY, t = 0.f, L = 0.f;
    for (int x = 0; x < kFewWarps; ++x) M = fmaxf(M, s_m[x][r]);
    for (int x = 0; x < kFewWarps; ++x) {
      const float f = ex2_from(s_m[x][r], M);
      t = fmaf(f, s_acc[x][r][d], t);
      L = fmaf(f, s_l[x][r], L);
    }
    if (a.nrel && d < D)
      for (int o = 0; o < a.nrel; ++o) t = fmaf(ex2_from(s_near[r][o], M), to_f(relv[o * D + d]), t);
    b_acc[r][d] = t;
    if (d == 0) {
      b_m[r] = M;
      b_l[r] = L;
    }
  }
  cl.sync();
  for (int e = rank * kFewWarps * 32 + threadIdx.x; e < R * DP; e += cs * kFewWarps * 32) {
    const int r = e / DP, d = e - r * DP;
    // All remote reads under way together: a block outside the cluster counts as this one with weight 0.
    float xm[kFewSplits], xl[kFewSplits], xa[kFewSplits], M = -INFINITY, t = 0.f, L = 0.f;
#pragma unroll
    for (int x = 0; x < kFewSplits; ++x) {
      const int from = x < cs ? x : rank;
      xm[x] = *cl.map_shared_rank(&b_m[r], from);
      xl[x] = *cl.map_shared_rank(&b_l[r], from);
      xa[x] = *cl.map_shared_rank(&b_acc[r][d], from);
    }
#pragma unroll
    for (int x = 0; x < kFewSplits; ++x) M = fmaxf(M, xm[x]);
#pragma unroll
    for (int x = 0; x < kFewSplits; ++x) {
      if (x >= cs) break;
      const float f = ex2_from(xm[x], M);
      t = fmaf(f, xa[x], t);
      L = fmaf(f, xl[x], L);
    }
    if (r >= rows) continue;
    const int i = r / g, h = hk * g + r % g;
    if (d < D)
      static_cast<T*>(a.o)[b * a.so.b + h * a.so.h + i * a.so.t + d] = from_f<T>(L == 0.f ? 0.f : t / L);
    if (d == 0 && a.lse)
      a.lse[((int64_t)b * a.H + h) * a.Tq + i] = L == 0.f ? -INFINITY : ((M == -INFINITY ? 0.f : M) + log2f(L)) * kLn2;
  }
  cl.sync();  // the block's sums have been read
}

template <typename T, int G, int R>
cudaError_t launch(const AttnArgs& a, cudaStream_t st) {
  // Splits: a block per SM, each with at least one full step of its groups.  Clusters of 16 start late (16
  // sequences of 128 keys a block: 8.6 -> 13.6 us), so each block has at least four steps there (one sequence, 16
  // heads of 64 over 4 key heads, 8192 keys: 20.5 -> 14.8 us).
  const int step = (sizeof(T) == 4 ? 2 : 4) * (32 / G) * kFewWarps;
  int cs = 1;
  while (cs < kFewSplits && (int64_t)a.B * a.Hkv * cs < 148 && cs * step * (cs < 8 ? 1 : 4) < a.Tk) cs *= 2;
  const int el = sizeof(T);
  const bool vec = attn_rows_aligned(a.q, a.sq, a.D, el) && attn_rows_aligned(a.k, a.sk, a.D, el) &&
                   attn_rows_aligned(a.v, a.sv, a.D, el) && a.D % 8 == 0;
  const size_t smem = (size_t)kFewStages * 2 * (sizeof(T) == 4 ? 2 : 4) * kFewWarps * 32 * 8 * sizeof(T);
  int regs;
  cudaError_t e = kernel_setup(attn_fwd_few<T, G, R>, smem, &regs);
  if (e == cudaSuccess && cs > 8)
    e = cudaFuncSetAttribute(attn_fwd_few<T, G, R>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cs, a.Hkv, a.B);
  cfg.blockDim = dim3(kFewWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cs;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attn_fwd_few<T, G, R>, a, cs, vec);
}

template <typename T, int G>
cudaError_t rows(const AttnArgs& a, cudaStream_t st) {
  const int n = a.Tq * (a.H / a.Hkv);
  if (n <= 1) return launch<T, G, 1>(a, st);
  if (n <= 2) return launch<T, G, 2>(a, st);
  return n <= 4 ? launch<T, G, 4>(a, st) : launch<T, G, 8>(a, st);
}

template <typename T>
cudaError_t width(const AttnArgs& a, cudaStream_t st) {
  if (a.D <= 32) return rows<T, 4>(a, st);
  return a.D <= 64 ? rows<T, 8>(a, st) : rows<T, 16>(a, st);
}

}  // namespace

cudaError_t attn_fwd_few_rows(const AttnArgs& a, cudaStream_t st) {
  if (a.ty == Ty::F32) return width<float>(a, st);
  return a.ty == Ty::F16 ? width<__half>(a, st) : width<__nv_bfloat16>(a, st);
}

}  // namespace gsv
