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
//             With a window, the near columns of P and dS become one more
//             operand each: dq += (near dS) relk, and the tile's share of
//             drelk = (near dS)^T q and drelv = (near P)^T do.
// That is 7 products for 5, the price of giving every gradient element one
// owner: no atomics, no fp32 copy of dq in memory, and bits that repeat.
//
// S and dP have two buffers: warp 8 issues the next tile's score products
// before it waits for this tile's operands.  Warps 0-3 and 4-7 take one half of
// a tile's columns each, one row per thread, which halves the time from scores
// to operands (alternate tiles per group: 2870 cycles a tile on the long causal
// case).  Warps 9 and 10 load tiles.
//
// Rounding: P and dS are rounded to the operands' type.  fp16 holds 2^-24 to
// 2^15 only, so P is carried as 2^15 P and dS with a power of two per head,
// the largest that no |dS| can overflow with (|dP - delta| <= 2 max|do|
// max|v|, norms taken by the row pass); both leave the fp32 sums at the end.
// Over many terms that rounding and the one of the result are alike, 1.41 times
// the latter together (measured 1.41 to 1.48 from 256 terms up, and up to 1.6
// below).  Sequences of up to kFineT therefore add what the operands' rounding
// lost as a second operand of each product (1.0 to 1.1 times): their launches
// wait more than they multiply, so it costs 1 to 7 % there against 14 to 18 %
// on long ones.  The near values always take both parts.
//
// Tiles come by TMA where rows are 16-byte vectors, else by cp.async (372
// against 670 us on the first case below).
//
// Measured on B200, bf16.  2 x 16 heads of 64, 4096 causal tokens: 330 us (and
// 25 for the row pass), 520 TFLOP/s of the five products, 730 of the seven; a
// key or query tile takes its softmax warps longer (two TMEM reads, one
// exponential and eight further operations a score, two stores) than the MMAs,
// which they wait for in turn (tensor pipe 34 % of the cycles, exponentials 40,
// issue slots 36).  16 utterances of up to 500 frames, 2 heads of
// 96, window 4: 25 us (12 for the rows, 3.6 for the relative sums); a block
// has 2 to 8 tiles there, so set-up, the first loads and the relative terms
// are half of it.
#include <algorithm>

#include "attn_launch.h"
#include "attn_tc.cuh"
#include "gsv_pdl.cuh"

namespace gsv {
namespace {

__device__ int g_give_ups;  // bounded waits of the kernels below that ran out in calls without a handle

constexpr int kBA = 128, kBB = 64;  // rows of the resident and of the streamed tiles
constexpr int kHalfB = kBB / 2;
constexpr int kFineT = 256;  // longest sequences with operands of twice the precision
constexpr int kThreads = 384;

template <int DP, bool REL>
struct BwdCfg {
  static constexpr int NC = (DP + 63) / 64;
  static constexpr uint32_t chunkA = kBA * 128, chunkB = kBB * 128, chunkR = 32 * 128;
  static constexpr uint32_t tileA = NC * chunkA, tileB = NC * chunkB;
  static constexpr int ST = NC == 2 && REL ? 3 : 4;
  static constexpr uint32_t rows = 2 * kBB * 4;  // nlse2 and ndelta of a streamed query tile
  static constexpr uint32_t rel = REL ? 2 * kBB * 32 * 4 : 0;  // its relative products (up to 31 offsets)
  static constexpr uint32_t stage = 2 * tileB;
  static constexpr uint32_t relk = REL ? NC * chunkR : 0;
  static constexpr uint32_t bandT = 2 * 32 * 128;  // 32 offsets x 128 rows in 16 bits, two chunks of 64 rows
  // keys: tables of ST stages; queries: the relative products of 128 rows.  The larger one.
  static constexpr uint32_t tables_k = ST * (rows + rel), tables_q = REL ? 2 * 32 * kBA * 4 : 0;
  static constexpr uint32_t tables = tables_k > tables_q ? tables_k : tables_q;
  static constexpr uint32_t smem = 2 * tileA + ST * stage + relk + tables;
};

struct BwdBars {
  uint64_t a_full, r_full, b_full[4], b_free[4], s_full[2], p_full[2], acc_full;
};

// A run of the workspace (16-byte aligned, a multiple of 16 bytes).
__device__ __forceinline__ void bulk_copy(uint32_t dst, const float* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// Tensor maps of the resident (128-row boxes) and the streamed tiles (64-row
// boxes); `on`: tiles come by TMA unless they hold rows behind a length, which
// must read as zeros: those come by cp.async.
struct BwdMaps {
  RowsMap qa, ka, va, ga, qb, kb, vb, gb;
  bool a_on, b_on;
};

// What the rounding of 32 values to an operand's 16 columns lost, as 16 more.
template <typename T>
__device__ __forceinline__ void store_lost(uint32_t taddr, uint32_t* packed, const float* x) {
#pragma unroll
  for (int c = 0; c < kHalfB; c += 2) {
    float lo, hi;
    lost2<T>(packed[c / 2], F2(x[c], x[c + 1])).get(lo, hi);
    packed[c / 2] = pack2<T>(lo, hi);
  }
  tmem_store16(taddr, packed);
}

// Adds the relative terms to the near scores and dP of a group's 32 columns, in
// TMEM, eight columns at a time (a rolled loop: inside the passes over all
// columns it would make those several times their size).  Column c has offset
// index d0 + step c; the warp's near columns are [begin, end).
template <typename F>
__device__ __forceinline__ void near_terms(uint32_t ts, int d0, int step, int begin, int end, int nrel, F add) {
  begin = max(0, begin);
  end = min(kHalfB, end);
  if (begin >= end) return;
#pragma unroll 1
  for (int c8 = begin & ~7; c8 < end; c8 += 8) {
    float x[8], y[8];
    tmem_load8(ts + c8, x);
    tmem_load8(ts + kBB + c8, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned r = (unsigned)(d0 + step * (c8 + e));
      if (r < (unsigned)nrel) add(c8 + e, r, x[e], y[e]);
    }
    uint32_t u[8], v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = __float_as_uint(x[e]), v[e] = __float_as_uint(y[e]);
    tmem_store8(ts + c8, u);
    tmem_store8(ts + kBB + c8, v);
  }
  tmem_store_wait();
}

template <typename T, int DP, bool REL>
__global__ void __launch_bounds__(kThreads, 1) attn_bwd_tc(const __grid_constant__ AttnArgs a,
                                                           const __grid_constant__ BwdWs ws,
                                                           const __grid_constant__ BwdMaps maps, const int nk,
                                                           const bool fine, const bool vec, const int ovec) {
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
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // The keys' blocks, which do more, come first; tiles slowest, the longest ones of a causal call first
  // (head by head, the two cases above took 17 and 2.6 us longer).
  const int D = a.D, g = a.H / a.Hkv, nq = cdiv(a.Tq, kBA), kblocks = nk * a.Hkv * a.B;
  const bool keys = (int)blockIdx.x < kblocks;
  const int unit = keys ? blockIdx.x : blockIdx.x - kblocks, hn = keys ? a.Hkv : a.H, tile = unit / (hn * a.B);
  const int b = (unit - tile * hn * a.B) / hn, head = unit % hn, hk = keys ? head : head / g;
  const int ql = clamp_len(a.qlen, b, a.Tq), kl = clamp_len(a.klen, b, a.Tk), off = kl - ql;
  static_assert(kBB == kRowBlock && kBA == 2 * kRowBlock, "a tile's row values are whole runs of the workspace");
  // First row of the resident tiles; streamed tiles of each head, and their number in all.
  const int r0 = (keys ? tile : nq - 1 - tile) * kBA;
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
  const int qfirst = first_query(ql, kl, a.causal);
  const int64_t bh0 = (int64_t)b * a.H + (keys ? hk * g : head);  // first head
  volatile int* abort = &s_abort;
  auto bar = [&](const uint64_t& m) { return smem_u32(&m); };

  if (threadIdx.x == 0) {
    s_abort = 0;
    mbar_init(bar(bars.a_full), 3);  // the announcement and the two loader warps
    mbar_init(bar(bars.r_full), 2);
    for (int s = 0; s < ST; ++s) {
      mbar_init(bar(bars.b_full[s]), 3);
      mbar_init(bar(bars.b_free[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar(bars.s_full[s]), 1);
      mbar_init(bar(bars.p_full[s]), 8);
    }
    mbar_init(bar(bars.acc_full), 1);
    fence_async_smem();
  }
  if (warp == 8) tmem_alloc(smem_u32(&s_tmem), 512);
  if (threadIdx.x == 9 * 32 && maps.a_on && maps.b_on) {
    prefetch_map(keys ? maps.ka : maps.qa);
    prefetch_map(keys ? maps.va : maps.ga);
    prefetch_map(keys ? maps.qb : maps.kb);
    prefetch_map(keys ? maps.gb : maps.vb);
  }
  pdl_wait();  // the row pass's values
  float gs = 1.f;  // the power of two that dS is carried with
  if (kHalf && nt > 0) {
    float nd = 0.f, nv = 0.f;
    for (int64_t x = threadIdx.x; x < (int64_t)heads * a.Tq; x += kThreads) nd = fmaxf(nd, ws.ndo[bh0 * a.Tq + x]);
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

  const uint32_t tRel = tS + ((nt + 1) & 1) * 2 * kBB;  // drelk, drelv: the scores of tile nt - 1

  if (warp >= 8) {
    if (nt > 0 && warp == 8) {
      constexpr uint32_t id_s = idesc_attn<T>(kBB, false), id_a = idesc_attn<T>(DP, true);
      const bool lead = elect_lane();
      const uint64_t dA0 = sdesc<64>(sA0), dA1 = sdesc<64>(sA1), dB = sdesc<64>(sB), mB = desc_mn(sB, C::chunkB);
      int fs = 0, fr = 0, us = 0;  // stage and round to fill from next, stage in use
      bool ok = warp_wait(bar(bars.a_full), 0, abort);
      auto scores = [&](int t) {
        ok = ok && warp_wait(bar(bars.b_full[fs]), fr & 1, abort);
        if (!ok) return;
        tc_fence_after();
        const uint32_t d = tS + (t & 1) * 2 * kBB, done = bar(bars.s_full[t & 1]);
        const uint64_t b0 = dB + fs * (C::stage >> 4);
        if (++fs == ST) fs = 0, ++fr;
        if (lead) {
          mma_rows<DP>(d, dA0, C::chunkA, b0, C::chunkB, id_s);
          mma_rows<DP>(d + kBB, dA1, C::chunkA, b0 + (C::tileB >> 4), C::chunkB, id_s);
          mma_commit(done);
        }
        __syncwarp();
      };
      scores(0);
      for (int t = 0; t < nt && ok; ++t) {
        if (t + 1 < nt) scores(t + 1);
        ok = ok && warp_wait(bar(bars.p_full[t & 1]), (t >> 1) & 1, abort);
        if (!ok) break;
        tc_fence_after();
        const uint32_t p = tS + (t & 1) * 2 * kBB, done = bar(bars.b_free[us]);
        const uint64_t m0 = mB + us * (C::stage >> 4), m1 = m0 + (C::tileB >> 4);
        if (++us == ST) us = 0;
        // Each group's 16 operand columns lie over the first half of its own scores, what their rounding
        // lost over the second.
        auto accumulate = [&](uint32_t acc, uint32_t op, uint64_t m, bool start) {
          if (start) mma_ts_first(acc, op, m, id_a);
          else mma_ts_acc(acc, op, m, id_a);
#pragma unroll
          for (int c = 1; c < kBB / 16; ++c)
            mma_ts_acc(acc, op + (c >> 1) * kHalfB + (c & 1) * 8, m + c * (2048 >> 4), id_a);
        };
        if (lead) {
          if (keys) accumulate(tAcc0, p, m1, t == 0);
          accumulate(tAcc1, p + kBB, m0, t == 0);
          if (fine) {
            if (keys) accumulate(tAcc0, p + 16, m1, false);
            accumulate(tAcc1, p + kBB + 16, m0, false);
          }
          mma_commit(done);
        }
        __syncwarp();
      }
      if (REL && !keys && ok) {
        // dq += (near ds) relk; the operand comes over the buffer of tile nt, in its order.
        ok = warp_wait(bar(bars.r_full), 0, abort) && warp_wait(bar(bars.p_full[nt & 1]), (nt >> 1) & 1, abort);
        tc_fence_after();
        if (ok && lead) {
          const int nrp = (a.nrel + 15) / 16 * 16;
          for (int x = 0; x < 2; ++x)
            for (int c = 0; c < nrp / 16; ++c)
              mma_ts_acc(tAcc1, tS + (nt & 1) * 2 * kBB + x * 16 + c * 8, desc_mn(sR + c * 2048, C::chunkR), id_a);
          // Rows of the result: 128 channels (those past the tile's are not read); columns: offsets.
          const uint32_t id_r = idesc_attn<T>(nrp, false) | (1u << 15);
          for (int x = 0; x < 4; ++x)  // ds and what its rounding lost, then p
            for (int c = 0; c < kBA / 16; ++c) {
              const uint64_t m = desc_mn((x >> 1 ? sA1 : sA0) + c * 2048, C::chunkA);
              const uint64_t d = sdesc<64>(sB + x * C::bandT + (c >> 2) * (C::bandT / 2) + (c & 3) * 32);
              if (x % 2 == 0 && c == 0) mma_bf16_first(tRel + (x >> 1) * 32, m, d, id_r);
              else mma_bf16_acc(tRel + (x >> 1) * 32, m, d, id_r);
            }
        }
      }
      if (lead) mma_commit(bar(bars.acc_full));
      if (!ok) *abort = 1;
      warp_wait(bar(bars.acc_full), 0, abort);  // nothing in flight when memory is given back
    } else if (nt > 0 && warp < 11) {
      const int tid = threadIdx.x - 9 * 32;
      Handover ho;
      bool ok = true;
      const T* q = static_cast<const T*>(a.q) + b * a.sq.b;
      const T* k = static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h;
      const T* v = static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h;
      const T* dout = static_cast<const T*>(a.dout) + b * a.sdo.b;
      // Per barrier: the first warp's lane 0 announces and issues what moves by bulk copies (full tiles,
      // row values); tails are copied by both warps, whose second arrival, or both, come when that is done.
      const bool first_warp = warp == 9;
      const bool full_a =
          maps.a_on && tma_fits(r0, kBA, keys ? kl : ql, keys ? a.Tk : a.Tq) && (keys || r0 >= qfirst);
      const uint32_t a_full = bar(bars.a_full);
      if (first_warp && lane == 0) {
        const uint32_t rel_bytes = REL && !keys ? 2u * 2 * kBB * a.nrel * 4 : 0;
        mbar_expect_tx(a_full, (full_a ? 2 * C::tileA : 0) + rel_bytes);
        if (full_a) {
          tma_tile<DP>(sA0, C::chunkA, keys ? maps.ka : maps.qa, a_full, r0, head, b);
          tma_tile<DP>(sA1, C::chunkA, keys ? maps.va : maps.ga, a_full, r0, head, b);
        }
        if (REL && !keys) bulk_copy(sTab, rel_at(ws, bh0, r0, a.nrel), rel_bytes, a_full);
      }
      if (!full_a) {
        if (keys) {
          load_tile<T, DP, kBA>(sA0, C::chunkA, k + (int64_t)r0 * a.sk.t, a.sk.t, kl - r0, D, vec, tid);
          load_tile<T, DP, kBA>(sA1, C::chunkA, v + (int64_t)r0 * a.sv.t, a.sv.t, kl - r0, D, vec, tid);
        } else {
          const int h = head;
          load_tile<T, DP, kBA>(sA0, C::chunkA, q + h * a.sq.h + (int64_t)r0 * a.sq.t, a.sq.t, ql - r0, D, vec, tid,
                                qfirst - r0);
          load_tile<T, DP, kBA>(sA1, C::chunkA, dout + h * a.sdo.h + (int64_t)r0 * a.sdo.t, a.sdo.t, ql - r0, D, vec,
                                tid, qfirst - r0);
        }
        ho.next(a_full);
      } else {
        warp_arrive(a_full);
      }
      if (REL && !keys) {  // needed last: a barrier of its own
        load_tile<T, DP, 32>(sR, C::chunkR, static_cast<const T*>(a.relk), D, a.nrel, D, vec, tid);
        ho.next(bar(bars.r_full));
      }
      int hh = 0, x = first, s = 0, round = 0;
      for (int t = 0; t < nt; ++t) {
        const int i0 = x * kBB;
        const uint32_t b0 = sB + s * C::stage, b1 = b0 + C::tileB, full = bar(bars.b_full[s]);
        if (round > 0) ok = ho.wait_free(bar(bars.b_free[s]), (round - 1) & 1, abort);
        if (!ok) break;
        const int h = keys ? hk * g + hh : hk;
        const bool whole =
            maps.b_on && tma_fits(i0, kBB, keys ? ql : kl, keys ? a.Tq : a.Tk) && (!keys || i0 >= qfirst);
        if (first_warp && lane == 0) {
          // Offsets of this pair of tiles: from r0 - (i0 + 63 + off) to r0 + 127 - (i0 + off).
          const bool near = REL && keys && r0 - (i0 + kBB - 1 + off) <= a.window &&
                            r0 + kBA - 1 - (i0 + off) >= -a.window;
          const uint32_t rel_bytes = near ? 2u * kBB * a.nrel * 4 : 0;
          mbar_expect_tx(full, (whole ? 2 * C::tileB : 0) + (keys ? C::rows : 0) + rel_bytes);
          if (whole) {
            tma_tile<DP>(b0, C::chunkB, keys ? maps.qb : maps.kb, full, i0, h, b);
            tma_tile<DP>(b1, C::chunkB, keys ? maps.gb : maps.vb, full, i0, h, b);
          }
          const uint32_t tab = sTab + s * (C::rows + C::rel);
          if (keys) bulk_copy(tab, row_at(ws, bh0 + hh, i0), C::rows, full);
          if (near) bulk_copy(tab + C::rows, rel_at(ws, bh0 + hh, i0, a.nrel), rel_bytes, full);
        }
        if (whole) {
          ho.flush();
          warp_arrive(full);
        } else {
          if (keys) {
            load_tile<T, DP, kBB>(b0, C::chunkB, q + h * a.sq.h + (int64_t)i0 * a.sq.t, a.sq.t, ql - i0, D, vec, tid,
                                  qfirst - i0);
            load_tile<T, DP, kBB>(b1, C::chunkB, dout + h * a.sdo.h + (int64_t)i0 * a.sdo.t, a.sdo.t, ql - i0, D, vec,
                                  tid, qfirst - i0);
          } else {
            load_tile<T, DP, kBB>(b0, C::chunkB, k + (int64_t)i0 * a.sk.t, a.sk.t, kl - i0, D, vec, tid);
            load_tile<T, DP, kBB>(b1, C::chunkB, v + (int64_t)i0 * a.sv.t, a.sv.t, kl - i0, D, vec, tid);
          }
          ho.next(full);
        }
        if (++s == ST) {
          s = 0;
          ++round;
        }
        if (++x == first + per) {
          x = first;
          ++hh;
        }
      }
      ho.flush();
      cp_wait<0>();
      if (!ok) *abort = 1;
    }
  } else {
    const int wg = warp >> 2, row = threadIdx.x & 127, own = r0 + row, c0 = wg * kHalfB;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;
    const float sl2 = a.scale * kLog2e, gp = gs * exp2f(-kShift);
    const F2 sl(sl2, sl2), gp2(gp, gp);
    bool ok = true;
    if (keys) {
      int x = first, st = 0, round = 0;  // streamed tile within its head; its stage
      for (int t = 0; t < nt; ++t) {
        ok = warp_wait(bar(bars.s_full[t & 1]), (t >> 1) & 1, abort);
        // The row values of the stage came with its tiles.
        ok = ok && warp_wait(bar(bars.b_full[st]), round & 1, abort);
        if (!ok) break;
        tc_fence_after();
        const int i0 = x * kBB + c0;  // query of this group's column 0
        if (++x == first + per) x = first;
        const float* tab = tables + st * ((C::rows + C::rel) / 4);
        if (++st == ST) st = 0, ++round;
        const float* nlse2 = tab + c0;
        const float* ndelta = tab + kBB + c0;
        const uint32_t tb = tS + (t & 1) * 2 * kBB + lanes;
        if (REL) {
          // Offset index of column 0; it falls by one per column and grows by one per row.
          const int d0 = own - (i0 + off) + a.window;
          const float* qrel = tab + 2 * kBB + c0 * a.nrel;
          near_terms(tb + c0, d0, -1, d0 - lane - a.nrel + 1, d0 - lane + 32, a.nrel, [&](int c, unsigned r, float& x, float& y) {
            x += qrel[c * a.nrel + r];
            y += qrel[(kBB + c) * a.nrel + r];
          });
        }
        float s[kHalfB], dp[kHalfB];
        tmem_load32(tb + c0, s);
        tmem_load32(tb + kBB + c0, dp);
        float p[kHalfB];
#pragma unroll
        for (int c = 0; c < kHalfB; c += 4) {
          const float4 L = *reinterpret_cast<const float4*>(nlse2 + c);
          fma2(F2(s[c], s[c + 1]), sl, F2(L.x, L.y)).get(p[c], p[c + 1]);
          fma2(F2(s[c + 2], s[c + 3]), sl, F2(L.z, L.w)).get(p[c + 2], p[c + 3]);
#pragma unroll
          for (int y = 0; y < 4; ++y) p[c + y] = ex2(p[c + y]);
        }
        const int skip = a.causal ? own - off - i0 : 0;  // columns before it do not see this key
        if (__any_sync(0xffffffffu, skip > 0)) {
#pragma unroll
          for (int c = 0; c < kHalfB; ++c)
            if (c < skip) p[c] = 0.f;
        }
        uint32_t p2[kHalfB / 2], d2[kHalfB / 2];
        float d[kHalfB];
#pragma unroll
        for (int c = 0; c < kHalfB; c += 4) {
          const float4 E = *reinterpret_cast<const float4*>(ndelta + c);
          F2 u = add2(F2(dp[c], dp[c + 1]), F2(E.x, E.y)), w = add2(F2(dp[c + 2], dp[c + 3]), F2(E.z, E.w));
          if (kHalf) u = mul2(u, gp2), w = mul2(w, gp2);
          mul2(u, F2(p[c], p[c + 1])).get(d[c], d[c + 1]);
          mul2(w, F2(p[c + 2], p[c + 3])).get(d[c + 2], d[c + 3]);
          p2[c / 2] = pack2<T>(p[c], p[c + 1]);
          p2[c / 2 + 1] = pack2<T>(p[c + 2], p[c + 3]);
          d2[c / 2] = pack2<T>(d[c], d[c + 1]);
          d2[c / 2 + 1] = pack2<T>(d[c + 2], d[c + 3]);
        }
        tmem_store16(tb + c0, p2);
        tmem_store16(tb + kBB + c0, d2);
        if (fine) {
          store_lost<T>(tb + c0 + 16, p2, p);
          store_lost<T>(tb + kBB + c0 + 16, d2, d);
        }
        tmem_store_wait();
        tc_fence_before();
        warp_arrive(bar(bars.p_full[t & 1]));
      }
    } else {
      const int n = allowed_keys(own, ql, kl, a.causal);
      const float* rw = row_at(ws, bh0, own);
      const float nlse2 = n > 0 ? rw[0] : -INFINITY, ndelta = n > 0 ? rw[kRowBlock] : 0.f;
      const F2 nl(nlse2, nlse2), nd(ndelta, ndelta);
      // This row's q . relk, then the near p as carried; do . relv, then the near ds as carried
      // (an odd pitch of nrel: no bank conflicts between rows).
      float* tq = tables + ((row / kBB) * 2 * kBB + row % kBB) * a.nrel;
      float* tg = tq + kBB * a.nrel;
      if (REL && nt > 0) ok = warp_wait(bar(bars.a_full), 0, abort);
      for (int t = 0; t < nt && ok; ++t) {
        ok = warp_wait(bar(bars.s_full[t & 1]), (t >> 1) & 1, abort);
        if (!ok) break;
        tc_fence_after();
        const int j0 = t * kBB + c0, lim = n - j0;
        const int d0 = j0 - (own + off) + a.window;
        const uint32_t tb = tS + (t & 1) * 2 * kBB + lanes;
        if (REL)  // the tables then hold the near scores and dp themselves
          near_terms(tb + c0, d0, 1, -(d0 + lane), a.nrel + 31 - (d0 + lane), a.nrel, [&](int, unsigned r, float& x, float& y) {
            x += tq[r];
            y += tg[r];
            tq[r] = x;
            tg[r] = y;
          });
        float s[kHalfB], dp[kHalfB];
        tmem_load32(tb + c0, s);
        tmem_load32(tb + kBB + c0, dp);
        float d[kHalfB];
#pragma unroll
        for (int c = 0; c < kHalfB; c += 2) {
          fma2(F2(s[c], s[c + 1]), sl, nl).get(s[c], s[c + 1]);
          s[c] = ex2(s[c]);
          s[c + 1] = ex2(s[c + 1]);
        }
        if (__any_sync(0xffffffffu, lim < kHalfB)) {
#pragma unroll
          for (int c = 0; c < kHalfB; ++c)
            if (c >= lim) s[c] = 0.f;
        }
        uint32_t d2[kHalfB / 2];
#pragma unroll
        for (int c = 0; c < kHalfB; c += 2) {
          F2 u = add2(F2(dp[c], dp[c + 1]), nd);
          if (kHalf) u = mul2(u, gp2);
          mul2(u, F2(s[c], s[c + 1])).get(d[c], d[c + 1]);
          d2[c / 2] = pack2<T>(d[c], d[c + 1]);
        }
        tmem_store16(tb + kBB + c0, d2);
        if (fine) store_lost<T>(tb + kBB + c0 + 16, d2, d);
        tmem_store_wait();
        tc_fence_before();
        warp_arrive(bar(bars.p_full[t & 1]));
      }
      if (REL && nt > 0) {
        asm volatile("bar.sync 1, 256;" ::: "memory");  // the near values of both groups are in the tables
        if (ok) {
          // Over the score columns of the buffer of tile nt, whose last readers were these warps.
          const int jb = own + off - a.window;
          // Their p (group 1) and ds (group 0) as operands over the rows, in the ring that the last MMAs have
          // read, and ds as dq's; each with a second operand of what its rounding lost.
          ok = warp_wait(bar(bars.b_free[(nt - 1) % ST]), ((nt - 1) / ST) & 1, abort);
          const uint32_t to = sB + wg * 2 * C::bandT + (row >> 6) * (C::bandT / 2) + (row & 7) * 2;
#pragma unroll 1
          for (int q0 = 0; q0 < a.nrel && ok; q0 += 16) {
            float d[16];
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int y = 0; y < 16; ++y) {
              const int r = q0 + y, j = jb + r;
              const bool in = r < a.nrel && j >= 0 && j < n;
              const float p = in ? ex2(fmaf(tq[in ? r : 0], sl2, nlse2)) : 0.f;
              d[y] = wg == 1 ? p : in ? p * ((tg[in ? r : 0] + ndelta) * (kHalf ? gp : 1.f)) : 0.f;
            }
#pragma unroll
            for (int y = 0; y < 16; y += 2) {
              hi[y / 2] = pack2<T>(d[y], d[y + 1]);
              float a0, a1;
              lost2<T>(hi[y / 2], F2(d[y], d[y + 1])).get(a0, a1);
              lo[y / 2] = pack2<T>(a0, a1);
            }
#pragma unroll
            for (int y = 0; y < 16; ++y) {
              const int r = q0 + y;
              if (r >= a.nrel) continue;
              const uint32_t at = to + r * 128 + ((((row & 63) >> 3) ^ (r & 7)) << 4);
              asm volatile("st.shared.b16 [%0], %1;" ::"r"(at), "h"((uint16_t)(hi[y / 2] >> (16 * (y & 1)))) : "memory");
              asm volatile("st.shared.b16 [%0], %1;" ::"r"(at + C::bandT), "h"((uint16_t)(lo[y / 2] >> (16 * (y & 1))))
                           : "memory");
            }
            if (wg == 0) {
              tmem_store8(tS + (nt & 1) * 2 * kBB + lanes + q0 / 2, hi);
              tmem_store8(tS + (nt & 1) * 2 * kBB + lanes + 16 + q0 / 2, lo);
            }
          }
          fence_async_smem();
          tmem_store_wait();
          tc_fence_before();
          if (ok) warp_arrive(bar(bars.p_full[nt & 1]));
        }
      }
    }
    if (nt > 0) ok = ok && warp_wait(bar(bars.acc_full), 0, abort);
    if (!ok) *abort = 1;
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
        T* out = static_cast<T*>(a.dq) + b * a.sdq.b + head * a.sdq.h + (int64_t)own * a.sdq.t;
#pragma unroll 1
        for (int c = wg * 32; c < DP; c += 64) {
          float o[32] = {};
          if (nt > 0) tmem_load32(tAcc1 + lanes + c, o);
          if (n == 0)
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = 0.f;
          if (own < a.Tq) store_row32<T>(out, c, D, ovec, o, inv);
        }
        if (REL) {
          // Lane = channel; group 0: drelk, group 1: drelv.
          const int64_t at = ((int64_t)b * a.H + head) * nq + r0 / kBA;
          float* part = ws.part + (at * 2 + wg) * a.nrel * D + row;
          const float f = wg == 0 ? inv : exp2f(-kShift);
          for (int q0 = 0; q0 < a.nrel; q0 += 16) {
            float v[16] = {};
            if (nt > 0) tmem_load16(tRel + wg * 32 + lanes + q0, v);
#pragma unroll
            for (int y = 0; y < 16; ++y)
              if (q0 + y < a.nrel && row < D) part[(int64_t)(q0 + y) * D] = v[y] * f;
          }
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (threadIdx.x == 0 && s_abort) give_up(a.err, &g_give_ups);
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
  const int ovec = std::min(store_mode(a.dq, a.sdq, a.D),
                            std::min(store_mode(a.dk, a.sdk, a.D), store_mode(a.dv, a.sdv, a.D)));
  const int nk = cdiv(a.Tk, kBA), nq = cdiv(a.Tq, kBA);
  const bool fine = std::max(a.Tq, a.Tk) <= kFineT;
  BwdMaps m = {};
  if (vec) {
    m.a_on = map_rows(&m.qa, a.q, a.ty, a.sq, a.B, a.H, a.Tq, a.D, kBA) &&
             map_rows(&m.ga, a.dout, a.ty, a.sdo, a.B, a.H, a.Tq, a.D, kBA) &&
             map_rows(&m.ka, a.k, a.ty, a.sk, a.B, a.Hkv, a.Tk, a.D, kBA) &&
             map_rows(&m.va, a.v, a.ty, a.sv, a.B, a.Hkv, a.Tk, a.D, kBA);
    m.b_on = map_rows(&m.qb, a.q, a.ty, a.sq, a.B, a.H, a.Tq, a.D, kBB) &&
             map_rows(&m.gb, a.dout, a.ty, a.sdo, a.B, a.H, a.Tq, a.D, kBB) &&
             map_rows(&m.kb, a.k, a.ty, a.sk, a.B, a.Hkv, a.Tk, a.D, kBB) &&
             map_rows(&m.vb, a.v, a.ty, a.sv, a.B, a.Hkv, a.Tk, a.D, kBB);
  }
  const PdlScope pdl(a.Tq > 0);  // its set-up runs beside the end of the row pass
  const unsigned blocks = (unsigned)(((int64_t)nk * a.Hkv + (int64_t)nq * a.H) * a.B);
  return launch_k(attn_bwd_tc<T, DP, REL>, blocks, kThreads, smem, st, a, ws, m, nk, fine, vec, ovec);
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

cudaError_t attn_bwd_give_ups(int* out, cudaStream_t st) { return read_give_ups(g_give_ups, out, st); }

}  // namespace gsv
