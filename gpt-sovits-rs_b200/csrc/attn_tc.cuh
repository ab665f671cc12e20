// attn_tc.cuh -- shared pieces of the tcgen05 attention kernels: TMEM loads and
// stores, descriptors, and the tile loader.
//
// Operand tiles live in shared memory as 64-channel chunks of 128-byte rows
// with the 128-byte swizzle (16-byte unit u of row r sits at unit u ^ (r & 7)).
// One such tile serves as a K-major operand (contraction over channels: q k^T)
// and as an MN-major one (contraction over rows: p v), so nothing is
// transposed or stored twice.
#pragma once
#include "attn_common.cuh"
#include "tc_common.cuh"

namespace gsv {
namespace {

__device__ __forceinline__ void tmem_load8(uint32_t taddr, float* v) {
  uint32_t r[8];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_load16(uint32_t taddr, float* v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_load32(uint32_t taddr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_load64(uint32_t taddr, float* v) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, "
      "%36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, "
      "%57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]),
        "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]),
        "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]),
        "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
        "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_store8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               :
               : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
      "%13, %14, %15, %16};"
               :
               : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
        "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}

__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
      "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
               :
               : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
        "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
        "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
               : "memory");
}

__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// MN-major operand tile, 128-byte swizzle: 8-row groups 1024 bytes apart,
// 64-channel chunks `chunk` bytes apart.
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t chunk) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(chunk >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}

// Instruction descriptor: fp32 accumulator, M = 128, operands of type T, B
// K-major or MN-major.
template <typename T>
__host__ __device__ constexpr uint32_t idesc_attn(int n, bool b_mn) {
  constexpr uint32_t f = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kM >> 4) << 24);
}

// D = A . B and D += A . B with A in TMEM (lane = row, two 16-bit values per
// column).  The accumulate flag is part of the instruction's form and the
// descriptors advance by constants, so that the issuing thread spends little
// between two MMAs.
__device__ __forceinline__ void mma_ts_first(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
  asm volatile("tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, 0;" ::"r"(d), "r"(a), "l"(b), "r"(idesc)
               : "memory");
}
__device__ __forceinline__ void mma_ts_acc(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
  asm volatile("tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, 1;" ::"r"(d), "r"(a), "l"(b), "r"(idesc)
               : "memory");
}

// D = A . B^T over DP channels of two K-major tiles (descriptors of their first
// chunk; chunks of chA and chB bytes).
template <int DP>
__device__ __forceinline__ void mma_rows(uint32_t d, uint64_t a, uint32_t chA, uint64_t b, uint32_t chB,
                                         uint32_t idesc) {
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
    const uint64_t da = a + (c >> 2) * (chA >> 4) + (c & 3) * 2, db = b + (c >> 2) * (chB >> 4) + (c & 3) * 2;
    if (c == 0) mma_bf16_first(d, da, db, idesc);
    else mma_bf16_acc(d, da, db, idesc);
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Two fp32 lanes per instruction.
struct F2 {
  unsigned long long v;
  F2() = default;
  __device__ __forceinline__ F2(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ void get(float& lo, float& hi) const {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
  }
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(a.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return a;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(a.v) : "l"(a.v), "l"(b.v));
  return a;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(a.v) : "l"(a.v), "l"(b.v));
  return a;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// What pack2's rounding of the two values lost.
template <typename T>
__device__ __forceinline__ F2 lost2(uint32_t packed, F2 x) {
  float lo, hi;
  if constexpr (std::is_same<T, __half>::value) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&packed));
    lo = f.x, hi = f.y;
  } else {
    lo = __uint_as_float(packed << 16), hi = __uint_as_float(packed & 0xffff0000u);
  }
  return fma2(F2(lo, hi), F2(-1.f, -1.f), x);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

constexpr int kLoaders = 64;  // threads that load tiles (two warps)

// ROWS x DP channels of a tile, from the global rows from .. valid - 1 of D
// channels; everything else is zero (rows left out may hold NaN, and 0 . NaN
// would reach the accumulators).  `vec`: rows are whole aligned 16-byte vectors and
// move by cp.async; else by single elements.  A chunk's 8 (or 4) units per row
// divide the 64 threads, so a thread keeps its unit and its swizzle and steps
// down the rows by one constant.
template <typename T, int DP, int ROWS>
__device__ __forceinline__ void load_tile(uint32_t dst, uint32_t chunk, const T* g, int64_t stride, int valid, int D,
                                          bool vec, int tid, int from = 0) {
  const unsigned span = max(valid - from, 0);
#pragma unroll
  for (int c = 0; c < (DP + 63) / 64; ++c) {
    constexpr int kFull = 8;
    const int units = DP - c * 64 >= 64 ? kFull : (DP - c * 64) / 8;
    const int step = kLoaders / units, u = tid % units, r0 = tid / units, col = c * 64 + u * 8;
    uint32_t a = dst + c * chunk + r0 * 128 + ((u ^ r0) & 7) * 16;
    const T* p = g + (int64_t)r0 * stride + col;
    const int64_t ps = (int64_t)step * stride;
    if (vec) {
      const bool in = col < D;
#pragma unroll 8
      for (int i = 0; i < ROWS / step; ++i, a += step * 128, p += ps) {
        const bool use = in && (unsigned)(r0 + i * step - from) < span;
        cp_async16(a, use ? p : g, use ? 16 : 0);
      }
    } else {
      for (int r = r0; r < ROWS; r += step, a += step * 128, p += ps) {
        uint32_t w[4] = {0u, 0u, 0u, 0u};
        if ((unsigned)(r - from) < span) {
          const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (col + i < D) w[i >> 1] |= (uint32_t)e[i] << (16 * (i & 1));
        }
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                     : "memory");
      }
    }
  }
}

__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// One arrival for a warp, after what its lanes did before (32 lanes arriving on
// one barrier are served one by one).
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// The loader warps' side of a full barrier: a tile's copies are handed over
// (completed, made visible to the tensor core, signalled) when the next tile's
// copies are under way, or before the loader has to block.
struct Handover {
  uint32_t bar = 0;
  __device__ __forceinline__ void flush() {
    if (!bar) return;
    cp_wait<0>();
    fence_async_smem();
    warp_arrive(bar);
    bar = 0;
  }
  __device__ __forceinline__ void next(uint32_t full) {
    cp_commit();
    if (bar) {
      cp_wait<1>();
      fence_async_smem();
      warp_arrive(bar);
    }
    bar = full;
  }
  __device__ __forceinline__ bool wait_free(uint32_t empty, uint32_t parity, volatile int* abort) {
    // A test that returns at once: a try_wait may sleep for microseconds with a tile not handed over.
    if (__all_sync(0xffffffffu, mbar_test(empty, parity))) return true;
    flush();
    return __all_sync(0xffffffffu, mbar_wait_fast(empty, parity, abort));
  }
};

// One lane of the warp, the same at every use.  The issuing warp runs its loop
// with all lanes and only the MMAs under this predicate, so that descriptors
// stay in uniform registers.
__device__ __forceinline__ bool elect_lane() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// A bounded wait of a whole warp, with one answer for all its lanes (the TMEM
// accesses after it need the warp together).
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xffffffffu, mbar_wait_fast(bar, parity, abort));
}

constexpr int kAttnCode = 17;  // error code of a give-up in a handle's word

// A bounded wait of the block gave up: said in the handle's word where the call
// has one, else counted.  The counts only grow, so that whoever reads one takes
// nothing from the others.  Called once, at a kernel's end: at each of the waits
// it made the long causal forward 1.6 % slower.
__device__ __forceinline__ void give_up(int* handle_word, int* count) {
  int abort;
  if (handle_word) raise_err(handle_word, &abort, kAttnCode);
  else atomicAdd(count, 1);
}

// Waits for the stream, then reads a count of give-ups.
cudaError_t read_give_ups(int& count, int* out, cudaStream_t st) {
  void* p = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&p, count);
  if (e == cudaSuccess) e = cudaMemcpyAsync(out, p, sizeof(int), cudaMemcpyDeviceToHost, st);
  return e == cudaSuccess ? cudaStreamSynchronize(st) : e;
}

// A [B][heads][T][D] tensor as a 4-D tensor map whose boxes are ROWS rows of a
// 64-channel chunk.  Axes of one element, or shared by broadcasting (stride 0),
// have extent 1 and coordinate 0.
struct RowsMap {
  CUtensorMap map;
  int mh, mb;  // 1: the axis is there
};

// False when the tensor cannot be mapped; its tiles then move by cp.async.
bool map_rows(RowsMap* m, const void* p, Ty ty, const Str3& s, int B, int heads, int T, int D, int rows) {
  if (T < 1 || (s.t <= 0 && T > 1) || !encode_fn()) return false;
  m->mh = heads > 1 && s.h != 0;
  m->mb = B > 1 && s.b != 0;
  const cuuint64_t pad = ((cuuint64_t)D * 2 + 15) / 16 * 16;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)T, (cuuint64_t)(m->mh ? heads : 1),
                              (cuuint64_t)(m->mb ? B : 1)};
  const cuuint64_t strides[3] = {T > 1 ? (cuuint64_t)s.t * 2 : pad, m->mh ? (cuuint64_t)s.h * 2 : pad,
                                 m->mb ? (cuuint64_t)s.b * 2 : pad};
  const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, es[4] = {1, 1, 1, 1};
  return encode_fn()(&m->map, ty == Ty::F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                     const_cast<void*>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether TMA gives a tile its zeros: all its rows are valid, or those that are
// not lie past the tensor's end, where TMA fills.
__device__ __forceinline__ bool tma_fits(int row, int rows, int valid, int T) {
  return row + rows <= valid || valid == T;
}

__device__ __forceinline__ void prefetch_map(const RowsMap& m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&m.map)) : "memory");
}

// One tile by TMA (one thread); its bytes count on `bar`.
template <int DP>
__device__ __forceinline__ void tma_tile(uint32_t dst, uint32_t chunk, const RowsMap& m, uint32_t bar, int row, int h,
                                         int b) {
#pragma unroll
  for (int c = 0; c < (DP + 63) / 64; ++c)
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst + c * chunk),
        "l"(reinterpret_cast<uint64_t>(&m.map)), "r"(bar), "r"(c * 64), "r"(row), "r"(h * m.mh), "r"(b * m.mb)
        : "memory");
}

// Cluster barrier (every thread of the cluster), and a read of another block's
// shared memory at the place of this block's `addr`.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float cluster_load(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// How rows of an output may be written: 0 by elements, 1 by 16-byte, 2 by
// 32-byte vectors (whole sectors per lane).
inline int store_mode(const void* p, const Str3& s, int D) {
  if (!attn_rows_aligned(p, s, D, 2)) return 0;
  const bool wide = reinterpret_cast<uintptr_t>(p) % 32 == 0 && s.b % 16 == 0 && s.h % 16 == 0 && s.t % 16 == 0;
  return wide && D % 16 == 0 ? 2 : 1;
}

// One row of 32 output channels starting at channel c, times f.
template <typename T>
__device__ __forceinline__ void store_row32(T* row, int c, int D, int mode, const float* v, float f) {
  if (mode) {
    uint4 u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      u[k].x = pack2<T>(v[8 * k] * f, v[8 * k + 1] * f);
      u[k].y = pack2<T>(v[8 * k + 2] * f, v[8 * k + 3] * f);
      u[k].z = pack2<T>(v[8 * k + 4] * f, v[8 * k + 5] * f);
      u[k].w = pack2<T>(v[8 * k + 6] * f, v[8 * k + 7] * f);
    }
    if (mode == 2) {
      if (c < D) st_global_v8(row + c, u[0], u[1]);
      if (c + 16 < D) st_global_v8(row + c + 16, u[2], u[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c + 8 * k < D) *reinterpret_cast<uint4*>(row + c + 8 * k) = u[k];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (c + i < D) row[c + i] = from_f<T>(v[i] * f);
  }
}

}  // namespace
}  // namespace gsv
