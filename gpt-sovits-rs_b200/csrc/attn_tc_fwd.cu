// attn_tc_fwd.cu -- attention forward on the tensor cores for fp16 and bf16
// (formulas in attn.h).
//
// A block of 8 warps takes 128 queries of one head and walks its key tiles of
// 128 with a running maximum and sum.  S = q k^T goes to TMEM (128 columns);
// warps 0-3 hold one query row per thread, turn S into P = exp2(s - m) and put
// it back in 16 bits, from where it is the A operand of O += P v (also
// in TMEM).  Warp 4 issues the MMAs, warps 5 and 6 load tiles.  TMEM (256
// columns) and shared memory are sized for two blocks per SM, so one block's
// softmax runs beside the other's MMAs.  Up to D = 64 the columns also hold P
// beside S: the next tile's scores are then computed while this tile's are
// being exponentiated.
//
// O is rescaled only when a row's maximum has grown by more than 2^8 since the
// scale in use was taken: P then stays below 2^8, which fp16 and bf16 hold
// with the same relative rounding, and most tiles skip the pass over O.
// P is rounded to the operands' type (the MMA takes no other); its row sum is
// taken in fp32 before that, so the rounding is unbiased noise of 2^-9 (bf16)
// or 2^-12 (fp16) of each term against one rounding of the same size at the
// output.
//
// Relative keys: q relk^T is one more small MMA ahead of the key tiles, kept as
// a table of 2 w + 1 values per row; the near scores replace their table entry
// when their tile comes by, and after the last tile their probabilities are
// one more P operand against the relative values' tile.
//
// Where the query tiles alone leave SMs idle, the blocks of a cluster deal out
// a query tile's key tiles among them and join their sums at the end, each
// block for its share of the rows, through distributed shared memory (rank
// order, one launch, no workspace).
//
// Tiles whose rows are 16-byte vectors come by TMA, others by cp.async, which
// took 13 % longer on the first case below.
//
// Measured on B200, bf16.  4 x 16 heads of 64, 4096 causal tokens: 198 us, 695
// TFLOP/s, 42 % of a large matrix product's rate.  The exponentials come first (16
// a cycle and SM, one per score: 120 us of that pipe, 64 % of its cycles), the
// two products take half of that (31 %); neither is full, because the softmax and
// the MMA warps wait for one another (issue slots 39 %).  A quarter of the
// exponentials as a polynomial took 15 us longer.  Blocks ordered head by head
// instead of the longest rows of all heads first: 219 us.  16 utterances of up to 500 frames, 2 heads
// of 96, window 4: 14.9 us, two thirds of it launch, first loads and the
// relative terms.
#include "attn_launch.h"
#include "attn_tc.cuh"

namespace gsv {
namespace {

__device__ int g_give_ups;  // bounded waits of the kernels below that ran out in calls without a handle

constexpr int kBM = 128, kBN = 128;
constexpr int kFwdThreads = 256;
constexpr int kSoftRegs = 176, kRestRegs = 80;  // 128 x 176 + 128 x 80 = 256 x 128

template <int DP>
struct FwdCfg {
  static constexpr int NC = (DP + 63) / 64;
  static constexpr uint32_t chunk = kBN * 128;     // bytes of a 64-channel chunk
  static constexpr uint32_t tile = NC * chunk;
  static constexpr int ST = NC == 1 ? 2 : 1;       // stages of the K and V rings
  static constexpr uint32_t smem = tile * (1 + 2 * ST);
  static constexpr bool own_p = DP <= 64;          // P beside S instead of over it
};

struct FwdBars {
  uint64_t q_full, k_full[2], k_free[2], v_full[2], v_free[2], s_full, s_free, p_full, o_full, pv_done;
};

// Tiles come by TMA (`on`) unless they hold rows behind a length, which must
// read as zeros: those come by cp.async.
struct FwdMaps {
  RowsMap q, k, v;
  bool q_on, kv_on;
};

template <typename T, int DP, bool REL>
__global__ void __launch_bounds__(kFwdThreads, 2) attn_fwd_tc(const __grid_constant__ AttnArgs a,
                                                              const __grid_constant__ FwdMaps maps, const int cs,
                                                              const bool vec, const int ovec) {
  using C = FwdCfg<DP>;
  constexpr int ST = C::ST;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ FwdBars bars;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ float s_m[kBM], s_l[kBM];  // for the other blocks of the cluster
  __shared__ float s_w[8][kBM / 2];
  const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u;
  const uint32_t sQ = base, sK = sQ + C::tile, sV = sK + ST * C::tile;
  float* tab = reinterpret_cast<float*>(smem_raw + (base - smem_u32(smem_raw)) + C::smem);  // [nrel][128]
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // Long rows of a causal mask first, of all heads, so that the last blocks are short ones.
  const int rank = blockIdx.x % cs, unit = blockIdx.x / cs, tile = unit / (a.H * a.B);
  const int i0 = (cdiv(a.Tq, kBM) - 1 - tile) * kBM, bh = unit - tile * a.H * a.B, b = bh / a.H, h = bh - b * a.H;
  const int ql = clamp_len(a.qlen, b, a.Tq), kl = clamp_len(a.klen, b, a.Tk), off = kl - ql;
  const int last = min(i0 + kBM, ql) - 1;
  const int kend = last < i0 ? 0 : allowed_keys(last, ql, kl, a.causal);
  // This block's key tiles: rank, rank + cs, ...
  const int all = (kend + kBN - 1) / kBN, nt = all > rank ? (all - rank + cs - 1) / cs : 0;
  const int hk = h / (a.H / a.Hkv), D = a.D;
  volatile int* abort = &s_abort;
  auto bar = [&](const uint64_t& m) { return smem_u32(&m); };

  if (threadIdx.x == 0) {
    s_abort = 0;
    mbar_init(bar(bars.q_full), 2);
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar(bars.k_full[s]), 2);
      mbar_init(bar(bars.v_full[s]), 2);
      mbar_init(bar(bars.k_free[s]), 1);
      mbar_init(bar(bars.v_free[s]), 1);
    }
    mbar_init(bar(bars.s_full), 1);
    mbar_init(bar(bars.p_full), 4);
    mbar_init(bar(bars.s_free), 4);
    mbar_init(bar(bars.o_full), 1);
    mbar_init(bar(bars.pv_done), 1);
    fence_async_smem();
  }
  if (warp == 4) tmem_alloc(smem_u32(&s_tmem), 256);
  if (threadIdx.x == 5 * 32 && maps.kv_on) {
    prefetch_map(maps.q);
    prefetch_map(maps.k);
    prefetch_map(maps.v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tS = s_tmem, tO = tS + kBN, tP = C::own_p ? tO + 64 : tS;
  const int nrp = REL ? (a.nrel + 15) / 16 * 16 : 0;

  if (warp >= 4) {
    reg_dec<kRestRegs>();
    if (nt > 0 && warp == 4) {
      constexpr uint32_t id_s = idesc_attn<T>(kBN, false), id_o = idesc_attn<T>(DP, true);
      const bool lead = elect_lane();
      const uint64_t dQ = sdesc<64>(sQ), dK = sdesc<64>(sK), mV = desc_mn(sV, C::chunk);
      bool ok = warp_wait(bar(bars.q_full), 0, abort);
      int kt = 0, vt = 0, pp = 0, sf = 0;
      auto scores = [&](uint32_t id) {  // S = q . (tile kt)^T
        const int s = kt % ST;
        ok = ok && warp_wait(bar(bars.k_full[s]), (kt / ST) & 1, abort);
        if (!ok) return;
        tc_fence_after();
        const uint64_t d = dK + s * (C::tile >> 4);
        const uint32_t kf = bar(bars.k_free[s]), sfull = bar(bars.s_full);
        if (lead) {
          mma_rows<DP>(tS, dQ, C::chunk, d, C::chunk, id);
          mma_commit(kf);
          mma_commit(sfull);
        }
        __syncwarp();
        ++kt;
      };
      auto scores_read = [&] {  // the softmax warps hold S in registers
        ok = ok && warp_wait(bar(bars.s_free), sf & 1, abort);
        ++sf;
        tc_fence_after();
      };
      auto values = [&](auto rows, bool first) {  // O (+)= P . (tile vt)
        const int s = vt % ST;
        ok = ok && warp_wait(bar(bars.v_full[s]), (vt / ST) & 1, abort);
        ok = ok && warp_wait(bar(bars.p_full), pp & 1, abort);
        ++pp;
        if (!ok) return;
        tc_fence_after();
        const uint64_t m = mV + s * (C::tile >> 4);
        const uint32_t vf = bar(bars.v_free[s]), done = bar(bars.pv_done);
        if (lead) {
          if (first) mma_ts_first(tO, tP, m, id_o);
          else mma_ts_acc(tO, tP, m, id_o);
#pragma unroll
          for (int c = 1; c < rows / 16; ++c) mma_ts_acc(tO, tP + c * 8, m + c * (2048 >> 4), id_o);
          mma_commit(vf);
          if (C::own_p) mma_commit(done);
        }
        __syncwarp();
        ++vt;
      };
      if (REL) {
        scores(idesc_attn<T>(nrp, false));
        scores_read();
      }
      if (C::own_p) scores(id_s);
      for (int t = 0; t < nt && ok; ++t) {
        if (C::own_p) {
          scores_read();
          if (t + 1 < nt) scores(id_s);
        } else {
          scores(id_s);
        }
        values(std::integral_constant<int, kBN>(), t == 0);
      }
      if (lead) mma_commit(bar(bars.o_full));
      int fin = 0;
      if (REL && ok) {
        values(nrp, false);
        if (lead) mma_commit(bar(bars.o_full));
        fin = 1;
      }
      if (!ok) *abort = 1;
      // Nothing of this block is in flight when its memory is given back.
      warp_wait(bar(bars.o_full), fin, abort);
    } else if (nt > 0 && warp < 7) {
      const int tid = threadIdx.x - 5 * 32;
      const T* q = static_cast<const T*>(a.q) + b * a.sq.b + h * a.sq.h;
      const T* k = static_cast<const T*>(a.k) + b * a.sk.b + hk * a.sk.h;
      const T* v = static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h;
      Handover ho;
      int kt = 0, vt = 0;
      bool ok = true;
      // Free stage of the K or V ring, or 0 when a wait gave up.
      auto stage = [&](bool is_k, int n) -> uint32_t {
        const int s = n % ST;
        if (n >= ST) ok = ho.wait_free(bar(is_k ? bars.k_free[s] : bars.v_free[s]), (n / ST - 1) & 1, abort);
        return ok ? (is_k ? sK : sV) + s * C::tile : 0;
      };
      // One tile: by TMA from the first loader warp, or by both warps' copies.
      auto fetch = [&](uint32_t dst, uint32_t full, bool on, const RowsMap& m, int head, const T* p, int64_t stride,
                       int row, int valid, int T_) {
        if (on && tma_fits(row, kBM, valid, T_)) {
          ho.flush();
          if (warp == 5) {
            if (lane == 0) {
              mbar_expect_tx(full, C::tile);
              tma_tile<DP>(dst, C::chunk, m, full, row, head, b);
            }
          } else {
            warp_arrive(full);
          }
        } else {
          load_tile<T, DP, kBM>(dst, C::chunk, p + (int64_t)row * stride, stride, valid - row, D, vec, tid);
          ho.next(full);
        }
      };
      fetch(sQ, bar(bars.q_full), maps.q_on, maps.q, h, q, a.sq.t, i0, ql, a.Tq);
      if (REL) {
        load_tile<T, DP, 32>(sK, C::chunk, static_cast<const T*>(a.relk), D, a.nrel, D, vec, tid);
        ho.next(bar(bars.k_full[kt++]));
      }
      for (int t = 0; t < nt && ok; ++t) {
        uint32_t dst = stage(true, kt);
        if (!dst) break;
        fetch(dst, bar(bars.k_full[kt++ % ST]), maps.kv_on, maps.k, hk, k, a.sk.t, (rank + t * cs) * kBN, kl, a.Tk);
        dst = stage(false, vt);
        if (!dst) break;
        fetch(dst, bar(bars.v_full[vt++ % ST]), maps.kv_on, maps.v, hk, v, a.sv.t, (rank + t * cs) * kBN, kl, a.Tk);
      }
      if (REL && ok) {
        const uint32_t dst = stage(false, vt);
        if (dst) {
          load_tile<T, DP, 32>(dst, C::chunk, static_cast<const T*>(a.relv), D, a.nrel, D, vec, tid);
          ho.next(bar(bars.v_full[vt % ST]));
        }
      }
      ho.flush();
      cp_wait<0>();
      if (!ok) *abort = 1;
    }
    if (cs > 1) {  // as the softmax warps join the cluster's sums
      cluster_sync();
      cluster_sync();
    }
  } else {
    reg_inc<kSoftRegs>();
    const int row = threadIdx.x, i = i0 + row;
    const int n = allowed_keys(i, ql, kl, a.causal);
    const uint32_t lanes = (uint32_t)warp << 21;
    const float sl2 = a.scale * kLog2e;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    int sp = 0;
    if (nt > 0) {
      if (REL) {
        ok = warp_wait(bar(bars.s_full), sp++ & 1, abort);
        tc_fence_after();
        if (ok)
          for (int r0 = 0; r0 < nrp; r0 += 16) {
            float v[16];
            tmem_load16(tS + lanes + r0, v);
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (r0 + r < a.nrel) tab[(r0 + r) * kBM + row] = v[r];
          }
        tc_fence_before();
        warp_arrive(bar(bars.s_free));
      }
      for (int t = 0; t < nt && ok; ++t) {
        ok = warp_wait(bar(bars.s_full), sp++ & 1, abort);
        if (!ok) break;
        tc_fence_after();
        const int j0 = (rank + t * cs) * kBN;
        if (REL) {
          // The near scores get their relative terms in TMEM, eight columns at a time (a rolled loop: the
          // same inside the pass below would make that several times its size for a few columns).
          // Offset index of column 0; it falls by one per row: the warp's near columns are [first, end).
          const int d0 = j0 - (i + off) + a.window;
          const int first = max(0, -(d0 + lane)), end = min(kBN, a.nrel + 31 - (d0 + lane));
          if (first < end) {
#pragma unroll 1
            for (int c8 = first & ~7; c8 < end; c8 += 8) {
              float x[8];
              tmem_load8(tS + lanes + c8, x);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const unsigned r = (unsigned)(d0 + c8 + e);
                if (r < (unsigned)a.nrel) {
                  x[e] += tab[r * kBM + row];
                  tab[r * kBM + row] = x[e];
                }
              }
              uint32_t u[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) u[e] = __float_as_uint(x[e]);
              tmem_store8(tS + lanes + c8, u);
            }
            tmem_store_wait();
          }
        }
        float s[kBN];
        tmem_load64(tS + lanes, s);
        tmem_load64(tS + lanes + 64, s + 64);
        if (C::own_p) {
          tc_fence_before();
          warp_arrive(bar(bars.s_free));
        }
        const int lim = n - j0;
        if (__any_sync(0xffffffffu, lim < kBN)) {
#pragma unroll
          for (int c = 0; c < kBN; ++c)
            if (c >= lim) s[c] = -INFINITY;
        }
        float m4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c < kBN - 4; c += 8)
#pragma unroll
          for (int x = 0; x < 4; ++x) m4[x] = max3(m4[x], s[c + x], s[c + 4 + x]);
#pragma unroll
        for (int x = 0; x < 4; ++x) m4[x] = fmaxf(m4[x], s[kBN - 4 + x]);
        const float mx = fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]);
        // The MMAs of the tile before have read P and added to O.
        if (C::own_p && t > 0) {
          ok = warp_wait(bar(bars.pv_done), (t - 1) & 1, abort);
          if (!ok) break;
          tc_fence_after();
        }
        // m is the maximum the scale in use was taken from; see the note on rescaling above.
        const bool grow = mx > m && (m == -INFINITY || (mx - m) * sl2 > 8.f);
        if (__any_sync(0xffffffffu, grow)) {
          const float mn = fmaxf(m, mx);
          const float alpha = m == -INFINITY ? 0.f : ex2((m - mn) * sl2);
          m = mn;
          l *= alpha;
          if (t > 0) {
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
              float o[32];
              tmem_load32(tO + lanes + c, o);
              uint32_t u[32];
#pragma unroll
              for (int x = 0; x < 32; ++x) u[x] = __float_as_uint(o[x] * alpha);
              tmem_store32(tO + lanes + c, u);
            }
          }
        }
        const float mu = m == -INFINITY ? 0.f : m * sl2;
        uint32_t p[kBN / 2];
        const F2 sl(sl2, sl2), nm(-mu, -mu);
        F2 la(0.f, 0.f), lb(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < kBN; c += 2) {
          float x, y;
          fma2(F2(s[c], s[c + 1]), sl, nm).get(x, y);
          x = ex2(x);
          y = ex2(y);
          if (c & 2) lb = add2(lb, F2(x, y));
          else la = add2(la, F2(x, y));
          p[c / 2] = pack2<T>(x, y);
        }
        float l0, l1;
        add2(la, lb).get(l0, l1);
        l += l0 + l1;
        tmem_store32(tP + lanes, p);
        tmem_store32(tP + lanes + 32, p + 32);
        tmem_store_wait();
        tc_fence_before();
        warp_arrive(bar(bars.p_full));
      }
      ok = ok && warp_wait(bar(bars.o_full), 0, abort);
      if (REL && ok) {
        tc_fence_after();
        const float mu = m == -INFINITY ? 0.f : m * sl2;
        const int base_j = i + off - a.window;
        for (int r0 = 0; r0 < nrp; r0 += 16) {
          float pr[16];
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            const int r = r0 + x, j = base_j + r;
            pr[x] = r < a.nrel && j >= 0 && j < n && ((j / kBN) & (cs - 1)) == rank ? ex2(fmaf(tab[r * kBM + row], sl2, -mu)) : 0.f;
          }
          uint32_t u[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) u[x] = pack2<T>(pr[2 * x], pr[2 * x + 1]);
          tmem_store8(tP + lanes + r0 / 2, u);
        }
        tmem_store_wait();
        tc_fence_before();
        warp_arrive(bar(bars.p_full));
        ok = warp_wait(bar(bars.o_full), 1, abort);
      }
      if (!ok) *abort = 1;
      tc_fence_after();
    }
    T* out = static_cast<T*>(a.o) + b * a.so.b + h * a.so.h;
    float* lse = a.lse ? a.lse + ((int64_t)b * a.H + h) * a.Tq : nullptr;
    if (cs == 1) {
      const bool some = nt > 0 && l != 0.f;
      const float inv = some ? 1.f / l : 0.f;
      if (ok && i < a.Tq && lse)
        lse[i] = some ? ((m == -INFINITY ? 0.f : m * sl2) + log2f(l)) * kLn2 : -INFINITY;
#pragma unroll 1
      for (int c = 0; c < DP; c += 32) {
        float o[32];
        if (nt > 0 && ok) tmem_load32(tO + lanes + c, o);
        if (!some)
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] = 0.f;
        if (ok && i < a.Tq) store_row32<T>(out + (int64_t)i * a.so.t, c, D, ovec, o, inv);
      }
    } else {
      // This block's sums as [row][channel] over the K and V rings, whose tiles have all been used;
      // the 16-byte unit u of a row sits at unit u ^ (row & 7), so that neither side has bank conflicts.
      const uint32_t sO = sK + row * DP * 4;
#pragma unroll 1
      for (int c = 0; c < DP; c += 32) {
        float o[32];
        if (nt > 0 && ok) tmem_load32(tO + lanes + c, o);
#pragma unroll
        for (int x = 0; x < 32; x += 4) {
          const uint32_t at = sO + (((c + x) / 4) ^ (row & 7)) * 16;
          asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(nt > 0 ? o[x] : 0.f),
                       "f"(nt > 0 ? o[x + 1] : 0.f), "f"(nt > 0 ? o[x + 2] : 0.f), "f"(nt > 0 ? o[x + 3] : 0.f)
                       : "memory");
        }
      }
      s_m[row] = nt > 0 ? m : -INFINITY;
      s_l[row] = nt > 0 ? l : 0.f;
      cluster_sync();
      // The weights of the blocks' sums in each row of this block's share.
      const int per = kBM / cs;
      if (row < per) {
        const int y = rank * per + row, iy = i0 + y;
        float w[8], v[8], M = -INFINITY, L = 0.f;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          w[x] = x < cs ? cluster_load(cluster_addr(smem_u32(s_m + y), x)) : -INFINITY;
          v[x] = x < cs ? cluster_load(cluster_addr(smem_u32(s_l + y), x)) : 0.f;
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) M = fmaxf(M, w[x]);
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          w[x] = w[x] == -INFINITY ? 0.f : ex2((w[x] - M) * sl2);
          L = fmaf(w[x], v[x], L);
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
        for (int x = 0; x < 8; ++x) s_w[x][row] = L == 0.f ? 0.f : w[x] * inv;
        if (iy < a.Tq && lse) lse[iy] = L == 0.f ? -INFINITY : ((M == -INFINITY ? 0.f : M * sl2) + log2f(L)) * kLn2;
      }
      asm volatile("bar.sync 1, 128;" ::: "memory");
      // 8 channels of a row per step, lanes side by side; two steps and two ranks under way together.
      constexpr int U = DP / 8;
      for (int e0 = row; e0 < per * U; e0 += 2 * kBM) {
        float o[2][8] = {};
        for (int x = 0; x < cs; x += 2) {
          float4 v[2][2][2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int e = min(e0 + j * kBM, per * U - 1), y = rank * per + e / U, u = e % U * 2;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const uint32_t from = cluster_addr(sK + y * DP * 4, x + k);
              v[j][k][0] = cluster_load4(from + (u ^ (y & 7)) * 16);
              v[j][k][1] = cluster_load4(from + ((u + 1) ^ (y & 7)) * 16);
            }
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int e = min(e0 + j * kBM, per * U - 1);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float f = s_w[x + k][e / U];
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                o[j][4 * q] = fmaf(f, v[j][k][q].x, o[j][4 * q]);
                o[j][4 * q + 1] = fmaf(f, v[j][k][q].y, o[j][4 * q + 1]);
                o[j][4 * q + 2] = fmaf(f, v[j][k][q].z, o[j][4 * q + 2]);
                o[j][4 * q + 3] = fmaf(f, v[j][k][q].w, o[j][4 * q + 3]);
              }
            }
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int e = e0 + j * kBM, iy = i0 + rank * per + e / U, c = e % U * 8;
          if (e >= per * U || iy >= a.Tq) continue;
          T* to = out + (int64_t)iy * a.so.t + c;
          if (ovec) {
            if (c < D) {
              uint4 u;
              u.x = pack2<T>(o[j][0], o[j][1]);
              u.y = pack2<T>(o[j][2], o[j][3]);
              u.z = pack2<T>(o[j][4], o[j][5]);
              u.w = pack2<T>(o[j][6], o[j][7]);
              *reinterpret_cast<uint4*>(to) = u;
            }
          } else {
#pragma unroll
            for (int y = 0; y < 8; ++y)
              if (c + y < D) to[y] = from_f<T>(o[j][y]);
          }
        }
      }
      cluster_sync();  // the sums have been read
    }
    tc_fence_before();
  }
  __syncthreads();
  if (threadIdx.x == 0 && s_abort) give_up(a.err, &g_give_ups);
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(s_tmem, 256);
  }
}

// A wait that runs out with nothing else in flight in its block.
__global__ void attn_wait_selftest_kernel(const __grid_constant__ AttnArgs a, const unsigned long long limit_ns) {
  __shared__ __align__(8) uint64_t s_bar;
  __shared__ int s_abort;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&s_bar), 1);
    s_abort = 0;
    fence_async_smem();
  }
  __syncthreads();
  if (threadIdx.x == 0 && !mbar_wait_fast(smem_u32(&s_bar), 0, &s_abort, limit_ns))
    give_up(a.err, &g_give_ups);
}

template <typename T, int DP, bool REL>
cudaError_t launch(const AttnArgs& a, cudaStream_t st) {
  const size_t smem = FwdCfg<DP>::smem + 1024 + (size_t)a.nrel * kBM * sizeof(float);
  int regs;
  cudaError_t e = kernel_setup(attn_fwd_tc<T, DP, REL>, smem, &regs);
  if (e != cudaSuccess) return e;
  const bool vec = attn_rows_aligned(a.q, a.sq, a.D, 2) && attn_rows_aligned(a.k, a.sk, a.D, 2) &&
                   attn_rows_aligned(a.v, a.sv, a.D, 2) && reinterpret_cast<uintptr_t>(a.relk) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(a.relv) % 16 == 0;
  const int ovec = store_mode(a.o, a.so, a.D);
  FwdMaps m = {};
  if (vec) {
    m.q_on = map_rows(&m.q, a.q, a.ty, a.sq, a.B, a.H, a.Tq, a.D, kBM);
    m.kv_on = map_rows(&m.k, a.k, a.ty, a.sk, a.B, a.Hkv, a.Tk, a.D, kBN) &&
              map_rows(&m.v, a.v, a.ty, a.sv, a.B, a.Hkv, a.Tk, a.D, kBN);
  }
  // Split while there are idle SMs; two blocks fit an SM, but sharing one pays only where each keeps 8 key tiles
  // (8 heads of 64, 1280 queries, 4096 keys: 39.6 -> 32.6 us; 9 utterances of 500, 2 heads of 96: 13.6 -> 25.1).
  // One utterance of 500 13.4 -> 12.3, 8 heads of 128 queries and 4096 keys 38.9 -> 14.1.
  const int nq = cdiv(a.Tq, kBM), nk = cdiv(a.Tk, kBN);
  int cs = 1;
  while (cs < 8 && 2 * cs <= nk && (int64_t)nq * a.H * a.B * 2 * cs <= sm_count() * (nk / (2 * cs) >= 8 ? 2 : 1)) cs *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)nq * a.H * a.B * cs));
  cfg.blockDim = dim3(kFwdThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cs;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cs > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, attn_fwd_tc<T, DP, REL>, a, m, cs, vec, ovec);
}

template <typename T, int DP>
cudaError_t rel(const AttnArgs& a, cudaStream_t st) {
  return a.nrel ? launch<T, DP, true>(a, st) : launch<T, DP, false>(a, st);
}

template <typename T>
cudaError_t width(const AttnArgs& a, cudaStream_t st) {
  if (a.D <= 32) return rel<T, 32>(a, st);
  if (a.D <= 64) return rel<T, 64>(a, st);
  return a.D <= 96 ? rel<T, 96>(a, st) : rel<T, 128>(a, st);
}

}  // namespace

cudaError_t attn_fwd_tensor(const AttnArgs& a, cudaStream_t st) {
  return a.ty == Ty::F16 ? width<__half>(a, st) : width<__nv_bfloat16>(a, st);
}

cudaError_t attn_wait_selftest(const AttnArgs& a, unsigned long long limit_ns, cudaStream_t st) {
  attn_wait_selftest_kernel<<<1, 32, 0, st>>>(a, limit_ns);
  return cudaGetLastError();
}

cudaError_t attn_fwd_give_ups(int* out, cudaStream_t st) { return read_give_ups(g_give_ups, out, st); }

}  // namespace gsv
