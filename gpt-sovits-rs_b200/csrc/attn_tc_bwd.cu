// attn_tc_bwd.cu -- attention backward on the tensor cores for fp16 and bf16
// (formulas in attn.h); the probabilities are recomputed from the saved
// log-sum-exp.
//
// One launch holds two kinds of blocks of one structure: a pair of 128-row
// tiles stays in shared memory, pairs of 64-row tiles stream past it.
//   keys:     k, v stay, q and do stream.  S^T = k q^T and dP^T = v do^T go to
//             TMEM; P^T and dS^T replace them in 16 bits and are the A
//             operands of dv += P^T do and dk += dS^T q.
//   queries:  q, do stay, k and v stream.  S = q k^T, dP = do v^T, and
//             dq += dS k.
// That is 7 products for 5, the price of giving every gradient element one
// owner: no atomics, no fp32 copy of dq in memory, and bits that repeat.
//
// S and dP have two buffers: warps 0-3 and 4-7 take alternate tiles (one row
// per thread), while warp 8 issues the next tile's score products before it
// waits for this tile's operands.  Warps 9 and 10 load tiles.
//
// Rounding: P and dS are rounded to the operands' type.  fp16 holds 2^-24 to
// 2^15 only, so P is carried as 2^15 P and dS with a power of two per head,
// the largest that no |dS| can overflow with (|dP - delta| <= 2 max|do|
// max|v|, norms taken by the row pass); both leave the fp32 sums at the end.
#include "attn_launch.h"
#include "attn_tc.cuh"

namespace gsv {
namespace {

__device__ int g_gave_up;  // set when a bounded wait of a kernel below ran out

constexpr int kBA = 128, kBB = 64;  // rows of the resident and of the streamed tiles
constexpr int kThreads = 384;

template <int DP, bool REL>
struct BwdCfg {
  static constexpr int NC = (DP + 63) / 64;
  static constexpr uint32_t chunkA = kBA * 128, chunkB = kBB * 128, chunkR = 32 * 128;
  static constexpr uint32_t tileA = NC * chunkA, tileB = NC * chunkB;
  static constexpr int ST = 3;
  static constexpr uint32_t rows = 2 * kBB * 4;  // lse2 and delta of a streamed query tile
  static constexpr uint32_t rel = REL ? 2 * kBB * 32 * 4 : 0;  // its relative products (up to 32 offsets)
  static constexpr uint32_t stage = 2 * tileB;
  static constexpr uint32_t relk = REL ? NC * chunkR : 0;
  // keys: tables of ST stages; queries: two [32][128] tables.  The larger one.
  static constexpr uint32_t tables_k = ST * (rows + rel), tables_q = REL ? 2 * 32 * kBA * 4 : 0;
  static constexpr uint32_t tables = tables_k > tables_q ? tables_k : tables_q;
  static constexpr uint32_t smem = 2 * tileA + ST * stage + relk + tables;
};

struct BwdBars {
  uint64_t a_full, b_full[3], b_free[3], s_full[2], p_full[2], acc_full;
};

__device__ __forceinline__ void cp_async4(uint32_t dst, const float* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}

template <typename T, int DP, bool REL>
__global__ void __launch_bounds__(kThreads, 1) attn_bwd_tc(const AttnArgs a, const BwdWs ws, const int nk,
                                                           const bool vec, const bool ovec) {
  using C = BwdCfg<DP, REL>;
  constexpr int ST = C::ST;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr float kShift = kHalf ? 15.f : 0.f;  // P is carried as 2^kShift P
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ BwdBars bars;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ float s_max[2][kThreads / 32];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023) & ~1023u;
  const uint32_t sA0 = base, sA1 = sA0 + C::tileA, sB = sA1 + C::tileA, sR = sB + ST * C::stage;
  float* tables = reinterpret_cast<float*>(smem_raw + (base - raw) + 2 * C::tileA + ST * C::stage + C::relk);
  const uint32_t sTab = smem_u32(tables);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, D = a.D, g = a.H / a.Hkv;
  const bool keys = (int)blockIdx.x < nk;
  if (keys && (int)blockIdx.y >= a.Hkv) return;
  const int hk = keys ? blockIdx.y : blockIdx.y / g;
  const int ql = clamp_len(a.qlen, b, a.Tq), kl = clamp_len(a.klen, b, a.Tk), off = kl - ql;
  // First row of the resident tiles; streamed tiles of each head, and their number in all.
  const int r0 = keys ? blockIdx.x * kBA : (int)(gridDim.x - 1 - blockIdx.x) * kBA;
  int first = 0, per = 0, heads = 1;
  if (keys) {
    heads = g;
    if (a.causal) first = max(0, r0 - off) / kBB;
    per = r0 < kl ? max(0, cdiv(ql, kBB) - first) : 0;
  } else {
    const int last = min(r0 + kBA, ql) - 1;
    per = last < r0 ? 0 : cdiv(allowed_keys(last, ql, kl, a.causal), kBB);
  }
  const int nt = per * heads;
  const int64_t row_h0 = ((int64_t)b * a.H + (keys ? hk * g : blockIdx.y)) * a.Tq;  // query row 0 of the first head
  volatile int* abort = &s_abort;
  auto bar = [&](const uint64_t& m) { return smem_u32(&m); };

  if (threadIdx.x == 0) {
    s_abort = 0;
    mbar_init(bar(bars.a_full), kLoaders);
    for (int s = 0; s < ST; ++s) {
      mbar_init(bar(bars.b_full[s]), kLoaders);
      mbar_init(bar(bars.b_free[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar(bars.s_full[s]), 1);
      mbar_init(bar(bars.p_full[s]), 128);
    }
    mbar_init(bar(bars.acc_full), 1);
    fence_async_smem();
  }
  if (warp == 8) tmem_alloc(smem_u32(&s_tmem), 512);
  float gs = 1.f;  // the power of two that dS is carried with
  if (kHalf && nt > 0) {
    float nd = 0.f, nv = 0.f;
    for (int64_t x = threadIdx.x; x < (int64_t)heads * a.Tq; x += kThreads) nd = fmaxf(nd, ws.ndo[row_h0 + x]);
    for (int x = threadIdx.x; x < kl; x += kThreads) nv = fmaxf(nv, ws.nv[((int64_t)b * a.Hkv + hk) * a.Tk + x]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      nd = fmaxf(nd, __shfl_xor_sync(0xffffffffu, nd, o));
      nv = fmaxf(nv, __shfl_xor_sync(0xffffffffu, nv, o));
    }
    if (lane == 0) {
      s_max[0][warp] = nd;
      s_max[1][warp] = nv;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (kHalf && nt > 0) {
    float nd = 0.f, nv = 0.f;
    for (int w = 0; w < kThreads / 32; ++w) {
      nd = fmaxf(nd, s_max[0][w]);
      nv = fmaxf(nv, s_max[1][w]);
    }
    const float most = 2.f * nd * nv;  // |dP - delta|
    // 2^14 / most rounded down to a power of two; rows without a finite positive bound stay as they are.
    if (most > 0.f && most < 1e30f) gs = exp2f(fminf(fmaxf(floorf(14.f - log2f(most)), -100.f), 100.f));
  }
  // TMEM columns: two buffers of (S, dP), then the accumulators.
  const uint32_t tS = s_tmem, tAcc0 = tS + 4 * kBB, tAcc1 = tAcc0 + DP;

  if (warp >= 8) {
    if (nt > 0 && warp == 8) {
      if (lane == 0) {
        constexpr uint32_t id_s = idesc_attn<T>(kBB, false), id_a = idesc_attn<T>(DP, true);
        bool ok = mbar_wait_fast(bar(bars.a_full), 0, abort);
        auto scores = [&](int t) {
          const int s = t % ST;
          ok = ok && mbar_wait_fast(bar(bars.b_full[s]), (t / ST) & 1, abort);
          if (!ok) return;
          tc_fence_after();
          const uint32_t d = tS + (t & 1) * 2 * kBB, b0 = sB + s * C::stage, b1 = b0 + C::tileB;
#pragma unroll
          for (int c = 0; c < DP / 16; ++c)
            mma_bf16(d, sdesc<64>(sA0 + (c >> 2) * C::chunkA + (c & 3) * 32),
                     sdesc<64>(b0 + (c >> 2) * C::chunkB + (c & 3) * 32), id_s, c > 0);
#pragma unroll
          for (int c = 0; c < DP / 16; ++c)
            mma_bf16(d + kBB, sdesc<64>(sA1 + (c >> 2) * C::chunkA + (c & 3) * 32),
                     sdesc<64>(b1 + (c >> 2) * C::chunkB + (c & 3) * 32), id_s, c > 0);
          mma_commit(bar(bars.s_full[t & 1]));
        };
        scores(0);
        for (int t = 0; t < nt && ok; ++t) {
          if (t + 1 < nt) scores(t + 1);
          const int s = t % ST;
          ok = ok && mbar_wait_fast(bar(bars.p_full[t & 1]), (t >> 1) & 1, abort);
          if (!ok) break;
          tc_fence_after();
          const uint32_t p = tS + (t & 1) * 2 * kBB, b0 = sB + s * C::stage, b1 = b0 + C::tileB;
          if (keys)
            for (int c = 0; c < kBB / 16; ++c)
              mma_ts(tAcc0, p + c * 8, desc_mn(b1 + c * 2048, C::chunkB), id_a, t > 0 || c > 0);
          for (int c = 0; c < kBB / 16; ++c)
            mma_ts(tAcc1, p + kBB + c * 8, desc_mn(b0 + c * 2048, C::chunkB), id_a, t > 0 || c > 0);
          mma_commit(bar(bars.b_free[s]));
        }
        if (REL && !keys && ok) {
          // dq += (near ds) relk; the operand comes over the buffer of tile nt, in its order.
          ok = mbar_wait_fast(bar(bars.p_full[nt & 1]), (nt >> 1) & 1, abort);
          tc_fence_after();
          if (ok)
            for (int c = 0; c < (a.nrel + 15) / 16; ++c)
              mma_ts(tAcc1, tS + (nt & 1) * 2 * kBB + c * 8, desc_mn(sR + c * 2048, C::chunkR), id_a, 1);
        }
        mma_commit(bar(bars.acc_full));
        if (!ok) raise_err(&g_gave_up, abort, 1);
        mbar_wait_fast(bar(bars.acc_full), 0, abort);  // nothing in flight when memory is given back
      }
      __syncwarp();
    } else if (nt > 0 && warp < 11) {
      const int tid = threadIdx.x - 9 * 32;
      Handover ho;
      bool ok = true;
      const T* q = static_cast<const T*>(a.q) + b * a.sq.b;
      const T* k = static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h;
      const T* v = static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h;
      const T* dout = static_cast<const T*>(a.dout) + b * a.sdo.b;
      if (keys) {
        load_tile<T, DP, kBA>(sA0, C::chunkA, k + (int64_t)r0 * a.sk.t, a.sk.t, kl - r0, D, vec, tid);
        load_tile<T, DP, kBA>(sA1, C::chunkA, v + (int64_t)r0 * a.sv.t, a.sv.t, kl - r0, D, vec, tid);
      } else {
        const int h = blockIdx.y;
        load_tile<T, DP, kBA>(sA0, C::chunkA, q + h * a.sq.h + (int64_t)r0 * a.sq.t, a.sq.t, ql - r0, D, vec, tid);
        load_tile<T, DP, kBA>(sA1, C::chunkA, dout + h * a.sdo.h + (int64_t)r0 * a.sdo.t, a.sdo.t, ql - r0, D, vec, tid);
        if (REL)
          load_tile<T, DP, 32>(sR, C::chunkR, static_cast<const T*>(a.relk), D, a.nrel, D, vec, tid);
      }
      ho.next(bar(bars.a_full));
      int hh = 0, x = first;
      for (int t = 0; t < nt; ++t) {
        const int s = t % ST, i0 = x * kBB;
        const uint32_t b0 = sB + s * C::stage, b1 = b0 + C::tileB;
        if (t >= ST) ok = ho.wait_free(bar(bars.b_free[s]), (t / ST - 1) & 1, abort);
        if (!ok) break;
        if (keys) {
          const int h = hk * g + hh;
          load_tile<T, DP, kBB>(b0, C::chunkB, q + h * a.sq.h + (int64_t)i0 * a.sq.t, a.sq.t, ql - i0, D, vec, tid);
          load_tile<T, DP, kBB>(b1, C::chunkB, dout + h * a.sdo.h + (int64_t)i0 * a.sdo.t, a.sdo.t, ql - i0, D, vec, tid);
          const int64_t row = row_h0 + (int64_t)hh * a.Tq + i0;
          const uint32_t tab = sTab + s * (C::rows + C::rel);
          for (int e = tid; e < 2 * kBB; e += kLoaders) {
            const int c = e & (kBB - 1);
            const bool in = i0 + c < a.Tq;
            cp_async4(tab + e * 4, (e < kBB ? ws.lse2 : ws.delta) + (in ? row + c : 0), in);
          }
          if (REL) {
            // Offsets of this pair of tiles: from r0 - (i0 + 63 + off) to r0 + 127 - (i0 + off).
            const int lo = r0 - (i0 + kBB - 1 + off), hi = r0 + kBA - 1 - (i0 + off);
            if (lo <= a.window && hi >= -a.window)
              for (int e = tid; e < kBB * a.nrel; e += kLoaders) {
                const bool in = i0 + e / a.nrel < a.Tq;
                const int64_t at = in ? row * a.nrel + e : 0;
                cp_async4(tab + C::rows + e * 4, ws.qrel + at, in);
                cp_async4(tab + C::rows + (kBB * 32 + e) * 4, ws.grel + at, in);
              }
          }
        } else {
          load_tile<T, DP, kBB>(b0, C::chunkB, k + (int64_t)i0 * a.sk.t, a.sk.t, kl - i0, D, vec, tid);
          load_tile<T, DP, kBB>(b1, C::chunkB, v + (int64_t)i0 * a.sv.t, a.sv.t, kl - i0, D, vec, tid);
        }
        ho.next(bar(bars.b_full[s]));
        if (++x == first + per) {
          x = first;
          ++hh;
        }
      }
      ho.flush();
      cp_wait<0>();
      if (!ok) raise_err(&g_gave_up, abort, 1);
    }
  } else {
    const int wg = warp >> 2, row = threadIdx.x & 127, own = r0 + row;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const float sl2 = a.scale * kLog2e, gp = gs * exp2f(-kShift);
    bool ok = true;
    if (keys) {
      int x = first + wg;  // streamed tile within its head
      for (int t = wg; t < nt && ok; t += 2, x += 2) {
        while (x >= first + per) x -= per;
        ok = warp_wait(bar(bars.s_full[wg]), (t >> 1) & 1, abort);
        // The tables of the stage: written by the loaders, who signalled b_full before the MMAs began.
        ok = ok && warp_wait(bar(bars.b_full[t % ST]), (t / ST) & 1, abort);
        if (!ok) break;
        tc_fence_after();
        const int i0 = x * kBB;
        const float* lse2 = tables + (t % ST) * ((C::rows + C::rel) / 4);
        const float* delta = lse2 + kBB;
        const float* qrel = lse2 + 2 * kBB;
        const float* grel = qrel + kBB * 32;
        const int d0 = own - (i0 + off) + a.window;       // offset index of column 0; falls by one per column
        const int skip = a.causal ? own - off - i0 : 0;   // columns before it do not see this key
        const bool near = REL && __any_sync(0xffffffffu, d0 >= 0 && d0 - (kBB - 1) < a.nrel);
        const bool cut = __any_sync(0xffffffffu, skip > 0);
        const uint32_t tb = tS + wg * 2 * kBB + lanes;
#pragma unroll 1
        for (int c0 = 0; c0 < kBB; c0 += 32) {
          float s[32], dp[32];
          tmem_load32(tb + c0, s);
          tmem_load32(tb + kBB + c0, dp);
          if (near) {
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const unsigned r = (unsigned)(d0 - c0 - c);
              if (r < (unsigned)a.nrel) {
                s[c] += qrel[(c0 + c) * a.nrel + r];
                dp[c] += grel[(c0 + c) * a.nrel + r];
              }
            }
          }
          uint32_t p2[16], d2[16];
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 L = *reinterpret_cast<const float4*>(lse2 + c0 + c);
            const float4 E = *reinterpret_cast<const float4*>(delta + c0 + c);
            const float l4[4] = {L.x, L.y, L.z, L.w}, e4[4] = {E.x, E.y, E.z, E.w};
            float p[4], d[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              p[y] = ex2(fmaf(s[c + y], sl2, kShift - l4[y]));
              if (cut && c0 + c + y < skip) p[y] = 0.f;
              d[y] = kHalf ? p[y] * (gp * (dp[c + y] - e4[y])) : p[y] * (dp[c + y] - e4[y]);
            }
            p2[c / 2] = pack2<T>(p[0], p[1]);
            p2[c / 2 + 1] = pack2<T>(p[2], p[3]);
            d2[c / 2] = pack2<T>(d[0], d[1]);
            d2[c / 2 + 1] = pack2<T>(d[2], d[3]);
          }
          tmem_store16(tb + c0 / 2, p2);
          tmem_store16(tb + kBB + c0 / 2, d2);
        }
        tmem_store_wait();
        tc_fence_before();
        mbar_arrive(bar(bars.p_full[wg]));
      }
    } else {
      const int n = allowed_keys(own, ql, kl, a.causal);
      const int64_t qrow = row_h0 + own;
      const float lse2 = n > 0 ? ws.lse2[qrow] : INFINITY, delta = n > 0 ? ws.delta[qrow] : 0.f;
      float* tq = tables;               // q . relk by offset, [nrel][128]
      float* tg = tables + 32 * kBA;    // do . relv, then the near ds
      if (REL && nt > 0) {
        for (int r = wg; r < a.nrel; r += 2) {
          tq[r * kBA + row] = n > 0 ? ws.qrel[qrow * a.nrel + r] : 0.f;
          tg[r * kBA + row] = n > 0 ? ws.grel[qrow * a.nrel + r] : 0.f;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
      for (int t = wg; t < nt && ok; t += 2) {
        ok = warp_wait(bar(bars.s_full[wg]), (t >> 1) & 1, abort);
        if (!ok) break;
        tc_fence_after();
        const int j0 = t * kBB, lim = n - j0;
        const int d0 = j0 - (own + off) + a.window;
        const bool near = REL && __any_sync(0xffffffffu, d0 < a.nrel && d0 + kBB > 0);
        const bool cut = __any_sync(0xffffffffu, lim < kBB);
        const uint32_t tb = tS + wg * 2 * kBB + lanes;
#pragma unroll 1
        for (int c0 = 0; c0 < kBB; c0 += 32) {
          float s[32], dp[32];
          tmem_load32(tb + c0, s);
          tmem_load32(tb + kBB + c0, dp);
          uint32_t d2[16];
          if (near) {
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              const unsigned r = (unsigned)(d0 + c0 + c);
              if (r < (unsigned)a.nrel) {
                s[c] += tq[r * kBA + row];
                dp[c] += tg[r * kBA + row];
              }
            }
          }
          float d[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            float p = ex2(fmaf(s[c], sl2, -lse2));
            if (cut && c0 + c >= lim) p = 0.f;
            d[c] = p * (dp[c] - delta);
            if (near) {
              const unsigned r = (unsigned)(d0 + c0 + c);
              if (r < (unsigned)a.nrel && c0 + c < lim) {
                ws.pband[qrow * a.nrel + r] = p;
                ws.sband[qrow * a.nrel + r] = d[c];
                tg[r * kBA + row] = d[c];
              }
            }
            if (kHalf) d[c] *= gs;
          }
#pragma unroll
          for (int c = 0; c < 32; c += 2) d2[c / 2] = pack2<T>(d[c], d[c + 1]);
          tmem_store16(tb + kBB + c0 / 2, d2);
        }
        tmem_store_wait();
        tc_fence_before();
        mbar_arrive(bar(bars.p_full[wg]));
      }
      if (REL && nt > 0) {
        asm volatile("bar.sync 1, 256;" ::: "memory");  // the near ds of both groups are in the table
        if (wg == (nt & 1) && ok) {
          // The score columns of the buffer: this group was their last reader.
          const int jb = own + off - a.window;
          for (int q0 = 0; q0 < a.nrel && ok; q0 += 16) {
            float d[16];
#pragma unroll
            for (int y = 0; y < 16; ++y) {
              const int r = q0 + y, j = jb + r;
              d[y] = r < a.nrel && j >= 0 && j < n ? tg[r * kBA + row] * gs : 0.f;
            }
            uint32_t u[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) u[y] = pack2<T>(d[2 * y], d[2 * y + 1]);
            tmem_store8(tS + wg * 2 * kBB + lanes + q0 / 2, u);
          }
          tmem_store_wait();
          tc_fence_before();
          if (ok) mbar_arrive(bar(bars.p_full[wg]));
        }
      }
    }
    if (nt > 0) ok = ok && warp_wait(bar(bars.acc_full), 0, abort);
    if (!ok) raise_err(&g_gave_up, abort, 1);
    tc_fence_after();
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      const float inv = a.scale / gs;
      if (keys) {
        // Group 0 writes dv, group 1 dk.
        T* out = wg == 0 ? static_cast<T*>(a.dv) + b * a.sdv.b + hk * a.sdv.h + (int64_t)own * a.sdv.t
                         : static_cast<T*>(a.dk) + b * a.sdk.b + hk * a.sdk.h + (int64_t)own * a.sdk.t;
        const float f = wg == 0 ? exp2f(-kShift) : inv;
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
          float o[32] = {};
          if (nt > 0) tmem_load32((wg == 0 ? tAcc0 : tAcc1) + lanes + c, o);
          if (own >= kl)
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = 0.f;
          if (own < a.Tk) store_row32<T>(out, c, D, ovec, o, f);
        }
      } else {
        const int n = allowed_keys(own, ql, kl, a.causal);
        T* out = static_cast<T*>(a.dq) + b * a.sdq.b + blockIdx.y * a.sdq.h + (int64_t)own * a.sdq.t;
#pragma unroll 1
        for (int c = wg * 32; c < DP; c += 64) {
          float o[32] = {};
          if (nt > 0) tmem_load32(tAcc1 + lanes + c, o);
          if (n == 0)
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = 0.f;
          if (own < a.Tq) store_row32<T>(out, c, D, ovec, o, inv);
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(s_tmem, 512);
  }
}

template <typename T, int DP, bool REL>
cudaError_t launch(const AttnArgs& a, const BwdWs& ws, cudaStream_t st) {
  const size_t smem = BwdCfg<DP, REL>::smem + 1024;
  int regs;
  cudaError_t e = kernel_setup(attn_bwd_tc<T, DP, REL>, smem, &regs);
  if (e != cudaSuccess) return e;
  const bool vec = attn_rows_aligned(a.q, a.sq, a.D, 2) && attn_rows_aligned(a.k, a.sk, a.D, 2) &&
                   attn_rows_aligned(a.v, a.sv, a.D, 2) && attn_rows_aligned(a.dout, a.sdo, a.D, 2) &&
                   reinterpret_cast<uintptr_t>(a.relk) % 16 == 0;
  const bool ovec = attn_rows_aligned(a.dq, a.sdq, a.D, 2) && attn_rows_aligned(a.dk, a.sdk, a.D, 2) &&
                    attn_rows_aligned(a.dv, a.sdv, a.D, 2);
  const int nk = cdiv(a.Tk, kBA), nq = cdiv(a.Tq, kBA);
  attn_bwd_tc<T, DP, REL><<<dim3(nk + nq, a.H, a.B), kThreads, smem, st>>>(a, ws, nk, vec, ovec);
  return cudaGetLastError();
}

template <typename T, int DP>
cudaError_t rel(const AttnArgs& a, const BwdWs& ws, cudaStream_t st) {
  return a.nrel ? launch<T, DP, true>(a, ws, st) : launch<T, DP, false>(a, ws, st);
}

template <typename T>
cudaError_t width(const AttnArgs& a, const BwdWs& ws, cudaStream_t st) {
  if (a.D <= 32) return rel<T, 32>(a, ws, st);
  if (a.D <= 64) return rel<T, 64>(a, ws, st);
  return a.D <= 96 ? rel<T, 96>(a, ws, st) : rel<T, 128>(a, ws, st);
}

}  // namespace

cudaError_t attn_bwd_tensor(const AttnArgs& a, const BwdWs& ws, cudaStream_t st) {
  return a.ty == Ty::F16 ? width<__half>(a, ws, st) : width<__nv_bfloat16>(a, ws, st);
}

cudaError_t attn_bwd_gave_up(int* out, cudaStream_t st) { return take_gave_up(g_gave_up, out, st); }

}  // namespace gsv
