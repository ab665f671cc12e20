// ops_api.cu -- C ABI of the attention and residual-norm operators
// (gsvdec_attention_*, gsvdec_norm_*): checks of arguments, then the launch.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <initializer_list>

#include "../../include/gsvdec.h"
#include "attn_launch.h"
#include "norm_grad.h"

namespace gsv {

int set_err(int code, const char* fmt, ...);  // gsvdec_api.cu

namespace {

constexpr int kMaxDevices = 64;

// GSV_OK when `device` is a device the kernels run on; looked up once each.
int device_ok(int device) {
  static std::atomic<int> known[kMaxDevices];  // 0 not looked up, 1 fine, else 2 + 16 major + minor
  int n = 0;
  if (device < 0 || device >= kMaxDevices || known[device].load(std::memory_order_acquire) == 0) {
    if (cudaGetDeviceCount(&n) != cudaSuccess || device < 0 || device >= n || device >= kMaxDevices) {
      cudaGetLastError();
      return set_err(GSV_E_INVALID_ARG, "device %d is not one of the %d CUDA devices", device, n);
    }
    int major = 0, minor = 0;
    cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
    cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, device);
    known[device].store(major == 10 && minor == 0 ? 1 : 2 + 16 * major + minor, std::memory_order_release);
  }
  const int k = known[device].load(std::memory_order_acquire);
  if (k == 1) return GSV_OK;
  return set_err(GSV_E_UNSUPPORTED, "device %d is sm_%d%d; the kernels are built for sm_100a", device, (k - 2) / 16,
                 (k - 2) % 16);
}

// The caller's current device is put back when the call returns.
struct OnDevice {
  int prev = -1;
  int rc;
  explicit OnDevice(int device) : rc(device_ok(device)) {
    if (rc != GSV_OK) return;
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != device) {
      const cudaError_t e = cudaSetDevice(device);
      if (e != cudaSuccess) rc = set_err(GSV_E_CUDA, "cudaSetDevice(%d): %s", device, cudaGetErrorString(e));
    } else {
      prev = -1;
    }
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

int finish(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return GSV_OK;
  cudaGetLastError();
  return set_err(GSV_E_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

Str3 str3(const int64_t* s) { return {s[0], s[1], s[2]}; }

// Whether no two elements of an output share an address: taken by increasing
// stride, each axis steps over everything the axes below it span.
bool spread(const int64_t* stride, const int* n, int axes, int64_t width) {
  int order[3] = {0, 1, 2};
  std::sort(order, order + axes, [&](int x, int y) { return stride[x] < stride[y]; });
  int64_t span = width;
  for (int i = 0; i < axes; ++i)
    if (n[i] == 0) return true;
  for (int i = 0; i < axes; ++i) {
    const int x = order[i];
    if (n[x] <= 1) continue;
    if (stride[x] < span) return false;
    span += stride[x] * (n[x] - 1);
  }
  return true;
}

// Whether every address is a multiple of the element's size (the kernels load
// whole elements; NULL counts as aligned).
bool elements_aligned(std::initializer_list<const void*> ps, int size) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % size) return false;
  return true;
}
bool forward_strides(const int64_t* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0) return false;
  return true;
}

int attn_shape(const gsvdec_attention* a, AttnArgs& o) {
  if (!a) return set_err(GSV_E_INVALID_ARG, "attention: NULL argument");
  if (a->dtype < GSV_DTYPE_F32 || a->dtype > GSV_DTYPE_BF16)
    return set_err(GSV_E_DTYPE, "attention: dtype %d is not one of F32, F16, BF16", a->dtype);
  if (a->B < 1 || a->B > 65535 || a->H < 1 || a->H > 65535 || a->Hkv < 1 || a->H % a->Hkv)
    return set_err(GSV_E_INVALID_ARG, "attention: B %d, H %d, Hkv %d (1 .. 65535, H a multiple of Hkv)", a->B, a->H,
                   a->Hkv);
  if ((int64_t)a->B * a->H > 1 << 24)  // heads times tiles is a launch's number of blocks
    return set_err(GSV_E_INVALID_ARG, "attention: B * H = %lld (up to 2^24)", (long long)a->B * a->H);
  if (a->Tq < 0 || a->Tk < 0 || a->Tq > (1 << 24) || a->Tk > (1 << 24))
    return set_err(GSV_E_INVALID_ARG, "attention: Tq %d, Tk %d (0 .. 2^24)", a->Tq, a->Tk);
  if (a->D < 1 || a->D > kAttnMaxD)
    return set_err(GSV_E_INVALID_ARG, "attention: D %d (1 .. %d)", a->D, kAttnMaxD);
  if (a->window < -1 || a->window > kAttnMaxWindow)
    return set_err(GSV_E_INVALID_ARG, "attention: window %d (-1 .. %d)", a->window, kAttnMaxWindow);
  if (a->causal != 0 && a->causal != 1) return set_err(GSV_E_INVALID_ARG, "attention: causal %d", a->causal);
  if (!(a->scale > 0.f) || !std::isfinite(a->scale))
    return set_err(GSV_E_INVALID_ARG, "attention: scale must be finite and positive");
  if (!forward_strides(a->q_stride, 3) || !forward_strides(a->k_stride, 3) || !forward_strides(a->v_stride, 3) ||
      !forward_strides(a->o_stride, 3) || !forward_strides(a->d_o_stride, 3))
    return set_err(GSV_E_INVALID_ARG, "attention: negative stride");
  o.ty = static_cast<Ty>(a->dtype);
  o.B = a->B;
  o.H = a->H;
  o.Hkv = a->Hkv;
  o.Tq = a->Tq;
  o.Tk = a->Tk;
  o.D = a->D;
  o.window = a->window;
  o.nrel = a->window >= 0 ? 2 * a->window + 1 : 0;
  o.causal = a->causal;
  o.scale = a->scale;
  o.q = a->q;
  o.k = a->k;
  o.v = a->v;
  o.relk = a->rel_k;
  o.relv = a->rel_v;
  o.dout = a->d_o;
  o.qlen = a->q_lengths;
  o.klen = a->k_lengths;
  o.o = a->o;
  o.dq = a->dq;
  o.dk = a->dk;
  o.dv = a->dv;
  o.drelk = a->drel_k;
  o.drelv = a->drel_v;
  o.lse = a->lse;
  o.sq = str3(a->q_stride);
  o.sk = str3(a->k_stride);
  o.sv = str3(a->v_stride);
  o.so = str3(a->o_stride);
  o.sdo = str3(a->d_o_stride);
  o.sdq = str3(a->dq_stride);
  o.sdk = str3(a->dk_stride);
  o.sdv = str3(a->dv_stride);
  o.ws = static_cast<char*>(a->workspace);
  o.ws_bytes = a->workspace_bytes;
  return GSV_OK;
}

int workspace_ok(const void* p, size_t have, size_t need, const char* what) {
  if (need == 0) return GSV_OK;
  if (!p || have < need || reinterpret_cast<uintptr_t>(p) % 16)
    return set_err(GSV_E_INVALID_ARG, "%s: workspace of %zu bytes given, %zu needed (16-byte aligned)", what, p ? have : 0,
                   need);
  return GSV_OK;
}

int attn_call(const gsvdec_attention* in, bool bwd, int device, void* stream) {
  AttnArgs a{};
  int rc = attn_shape(in, a);
  if (rc != GSV_OK) return rc;
  const bool q = a.Tq > 0, k = a.Tk > 0;
  if ((q && (!a.q || !a.o)) || (k && (!a.k || !a.v)))
    return set_err(GSV_E_INVALID_ARG, "attention: q, k, v or o is NULL");
  if (a.nrel && (!a.relk || !a.relv)) return set_err(GSV_E_INVALID_ARG, "attention: a window needs rel_k and rel_v");
  const int el = a.ty == Ty::F32 ? 4 : 2;
  if (!elements_aligned({a.q, a.k, a.v, a.relk, a.relv, a.o}, el) || !elements_aligned({a.lse, a.qlen, a.klen}, 4) ||
      (bwd && !elements_aligned({a.dout, a.dq, a.dk, a.dv, a.drelk, a.drelv}, el)))
    return set_err(GSV_E_INVALID_ARG, "attention: a tensor is not aligned to its elements");
  const int nq[3] = {a.B, a.H, a.Tq}, nk[3] = {a.B, a.Hkv, a.Tk};
  if (!bwd && !spread(in->o_stride, nq, 3, a.D))
    return set_err(GSV_E_INVALID_ARG, "attention: the rows of o overlap");
  if (bwd) {
    if ((q && (!a.dout || !a.dq || !a.lse)) || (k && (!a.dk || !a.dv)))
      return set_err(GSV_E_INVALID_ARG, "attention: d_o, lse, dq, dk or dv is NULL");
    if (a.nrel && (!a.drelk || !a.drelv))
      return set_err(GSV_E_INVALID_ARG, "attention: a window needs drel_k and drel_v");
    if (!spread(in->dq_stride, nq, 3, a.D) || !spread(in->dk_stride, nk, 3, a.D) || !spread(in->dv_stride, nk, 3, a.D))
      return set_err(GSV_E_INVALID_ARG, "attention: the rows of dq, dk or dv overlap");
  }
  if (attn_most_blocks(a, bwd) > INT32_MAX)
    return set_err(GSV_E_INVALID_ARG, "attention: %lld tiles of rows are more than a launch's blocks (2^31 - 1)",
                   (long long)attn_most_blocks(a, bwd));
  rc = workspace_ok(a.ws, a.ws_bytes, bwd ? attn_bwd_workspace(a) : attn_fwd_workspace(a), "attention");
  if (rc != GSV_OK) return rc;
  OnDevice dev(device);
  if (dev.rc != GSV_OK) return dev.rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return bwd ? finish(attn_backward(a, st), "attention backward") : finish(attn_forward(a, st), "attention forward");
}

int norm_shape(const gsvdec_norm* a, NormArgs& o) {
  if (!a) return set_err(GSV_E_INVALID_ARG, "norm: NULL argument");
  if (a->dtype < GSV_DTYPE_F32 || a->dtype > GSV_DTYPE_BF16)
    return set_err(GSV_E_DTYPE, "norm: dtype %d is not one of F32, F16, BF16", a->dtype);
  if (a->layout != GSV_LAYOUT_BCT && a->layout != GSV_LAYOUT_BTC)
    return set_err(GSV_E_INVALID_ARG, "norm: layout %d", a->layout);
  const int most = a->layout == GSV_LAYOUT_BTC ? kNormRowsMaxC : kNormTimeMaxC;
  if (a->B < 1 || a->T < 0 || a->C < 1 || a->C > most || (int64_t)a->B * a->T > (1ll << 28))
    return set_err(GSV_E_INVALID_ARG, "norm: B %d, C %d (1 .. %d), T %d (B T up to 2^28)", a->B, a->C, most, a->T);
  if (!(a->eps >= 0.f) || !std::isfinite(a->eps))
    return set_err(GSV_E_INVALID_ARG, "norm: eps must be finite and not negative");
  if (!forward_strides(a->x_stride, 2) || !forward_strides(a->y_stride, 2) || !forward_strides(a->d_out_stride, 2))
    return set_err(GSV_E_INVALID_ARG, "norm: negative stride");
  o.ty = static_cast<Ty>(a->dtype);
  o.rows = a->layout == GSV_LAYOUT_BTC;
  o.B = a->B;
  o.C = a->C;
  o.T = a->T;
  o.eps = a->eps;
  o.x = {a->x, a->x_stride[0], a->x_stride[1]};
  o.y = {a->y, a->y_stride[0], a->y_stride[1]};
  o.out = {a->out, a->out_stride[0], a->out_stride[1]};
  o.dout = {a->d_out, a->d_out_stride[0], a->d_out_stride[1]};
  o.dx = {a->dx, a->dx_stride[0], a->dx_stride[1]};
  o.gamma = a->gamma;
  o.beta = a->beta;
  o.mean = a->mean;
  o.rstd = a->rstd;
  o.len = a->lengths;
  o.dgamma = a->dgamma;
  o.dbeta = a->dbeta;
  o.part = static_cast<float*>(a->workspace);
  o.ws_bytes = a->workspace_bytes;
  return GSV_OK;
}

int norm_call(const gsvdec_norm* in, bool bwd, int device, void* stream) {
  NormArgs a{};
  int rc = norm_shape(in, a);
  if (rc != GSV_OK) return rc;
  const bool any = a.T > 0;
  if (!a.gamma || (any && (!a.x.p || !a.mean || !a.rstd)))
    return set_err(GSV_E_INVALID_ARG, "norm: x, gamma, mean or rstd is NULL");
  const int el = a.ty == Ty::F32 ? 4 : 2;
  if (!elements_aligned({a.x.p, a.y.p}, el) || !elements_aligned({a.gamma, a.mean, a.rstd, a.len}, 4) ||
      (bwd ? !elements_aligned({a.dout.p, a.dx.p}, el) || !elements_aligned({a.dgamma, a.dbeta}, 4)
           : !elements_aligned({a.out.p}, el) || !elements_aligned({a.beta}, 4)))
    return set_err(GSV_E_INVALID_ARG, "norm: a tensor is not aligned to its elements");
  const int64_t* s = bwd ? in->dx_stride : in->out_stride;
  const int inner = a.rows ? a.C : a.T, n[2] = {a.B, a.rows ? a.T : a.C};
  if (any && !spread(s, n, 2, inner))
    return set_err(GSV_E_INVALID_ARG, "norm: the rows of %s overlap", bwd ? "dx" : "out");
  if (!bwd && (!a.beta || (any && !a.out.p))) return set_err(GSV_E_INVALID_ARG, "norm: beta or out is NULL");
  if (bwd && (!a.dgamma || !a.dbeta || (any && (!a.dout.p || !a.dx.p))))
    return set_err(GSV_E_INVALID_ARG, "norm: d_out, dx, dgamma or dbeta is NULL");
  if (bwd) {
    rc = workspace_ok(a.part, a.ws_bytes, norm_bwd_workspace(a), "norm");
    if (rc != GSV_OK) return rc;
  }
  OnDevice dev(device);
  if (dev.rc != GSV_OK) return dev.rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return bwd ? finish(norm_backward(a, st), "norm backward") : finish(norm_forward(a, st), "norm forward");
}

}  // namespace

// gsvdec_selftest_attention_wait without a handle.
int ops_wait_selftest(int device, unsigned long long limit_ns, cudaStream_t st) {
  OnDevice dev(device);
  if (dev.rc != GSV_OK) return dev.rc;
  return finish(attn_wait_selftest(AttnArgs{}, limit_ns, st), "attention wait self-test");
}

}  // namespace gsv

extern "C" {

int gsvdec_attention_workspace(const gsvdec_attention* a, int backward, size_t* bytes) {
  if (!bytes) return gsv::set_err(GSV_E_INVALID_ARG, "attention: NULL argument");
  gsv::AttnArgs o{};
  const int rc = gsv::attn_shape(a, o);
  if (rc != GSV_OK) return rc;
  *bytes = backward ? gsv::attn_bwd_workspace(o) : gsv::attn_fwd_workspace(o);
  return GSV_OK;
}

int gsvdec_attention_forward(const gsvdec_attention* a, int device, void* stream) {
  return gsv::attn_call(a, false, device, stream);
}

int gsvdec_attention_backward(const gsvdec_attention* a, int device, void* stream) {
  return gsv::attn_call(a, true, device, stream);
}

int gsvdec_ops_status(int device, void* stream) {
  gsv::OnDevice dev(device);
  if (dev.rc != GSV_OK) return dev.rc;
  // What this thread has been told of; the counts themselves belong to all threads.
  thread_local int seen[gsv::kMaxDevices][3] = {};
  int now[3] = {};
  cudaError_t e = gsv::attn_fwd_give_ups(&now[0], static_cast<cudaStream_t>(stream));
  if (e == cudaSuccess) e = gsv::attn_bwd_give_ups(&now[1], static_cast<cudaStream_t>(stream));
  if (e == cudaSuccess) e = gsv::norm_give_ups(&now[2], static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return gsv::finish(e, "operator status");
  if (std::equal(now, now + 3, seen[device])) return GSV_OK;
  std::copy(now, now + 3, seen[device]);
  return gsv::set_err(GSV_E_TIMEOUT, "a bounded device wait of an operator on device %d gave up", device);
}

int gsvdec_norm_workspace(const gsvdec_norm* a, size_t* bytes) {
  if (!bytes) return gsv::set_err(GSV_E_INVALID_ARG, "norm: NULL argument");
  gsv::NormArgs o{};
  const int rc = gsv::norm_shape(a, o);
  if (rc != GSV_OK) return rc;
  *bytes = gsv::norm_bwd_workspace(o);
  return GSV_OK;
}

int gsvdec_norm_forward(const gsvdec_norm* a, int device, void* stream) {
  return gsv::norm_call(a, false, device, stream);
}

int gsvdec_norm_backward(const gsvdec_norm* a, int device, void* stream) {
  return gsv::norm_call(a, true, device, stream);
}

}  // extern "C"
