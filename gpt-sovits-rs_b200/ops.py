"""Attention and residual norm of the text encoder with their gradients, on CUDA tensors.

Stand-alone operators over ``gsvdec_attention_*`` and ``gsvdec_norm_*``
(include/gsvdec.h): no handle and no state.  Each call runs on the current
stream of its tensors' device, takes outputs and workspace from torch's
allocator, does not synchronise and can be captured in a CUDA graph.  The
forward calls return what their backward needs; autograd does not record them
(a torch.autograd.Function of a forward and its backward makes them trainable).
"""
from __future__ import annotations

import ctypes
import functools
import math
import struct
from typing import Optional

_I64x3 = ctypes.c_int64 * 3
_I64x2 = ctypes.c_int64 * 2
_vp = ctypes.c_void_p


class _Attention(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_int) for n in ("dtype", "B", "H", "Hkv", "Tq", "Tk", "D", "window", "causal")]
                + [("scale", ctypes.c_float), ("q_lengths", _vp), ("k_lengths", _vp), ("q", _vp), ("k", _vp),
                   ("v", _vp), ("q_stride", _I64x3), ("k_stride", _I64x3), ("v_stride", _I64x3), ("rel_k", _vp),
                   ("rel_v", _vp), ("o", _vp), ("o_stride", _I64x3), ("lse", _vp), ("d_o", _vp),
                   ("d_o_stride", _I64x3), ("dq", _vp), ("dk", _vp), ("dv", _vp), ("dq_stride", _I64x3),
                   ("dk_stride", _I64x3), ("dv_stride", _I64x3), ("drel_k", _vp), ("drel_v", _vp),
                   ("workspace", _vp), ("workspace_bytes", ctypes.c_size_t)])


class _Norm(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_int) for n in ("dtype", "layout", "B", "C", "T")]
                + [("eps", ctypes.c_float), ("lengths", _vp), ("x", _vp), ("y", _vp), ("x_stride", _I64x2),
                   ("y_stride", _I64x2), ("gamma", _vp), ("beta", _vp), ("mean", _vp), ("rstd", _vp), ("out", _vp),
                   ("out_stride", _I64x2), ("d_out", _vp), ("dx", _vp), ("d_out_stride", _I64x2),
                   ("dx_stride", _I64x2), ("dgamma", _vp), ("dbeta", _vp), ("workspace", _vp),
                   ("workspace_bytes", ctypes.c_size_t)])


LAYOUTS = {"bct": 0, "btc": 1}

# The two argument structures, packed in one go (setting ctypes fields one by
# one costs more than the smallest call's kernel).
_ATTENTION = struct.Struct("@9if" + "2q3q9q2qq3qq" + "q3q3q9q2q" + "qQ")
_NORM = struct.Struct("@5if" + "qqq2q2qqqqqq2q" + "qq2q2qqq" + "qQ")
assert _ATTENTION.size == ctypes.sizeof(_Attention) and _NORM.size == ctypes.sizeof(_Norm)
_Z3 = (0, 0, 0)


def declare(lib) -> None:
    """Argument types of the operators' C functions."""
    sz = ctypes.POINTER(ctypes.c_size_t)
    lib.gsvdec_attention_workspace.argtypes = [_vp, ctypes.c_int, sz]
    lib.gsvdec_attention_forward.argtypes = [_vp, ctypes.c_int, _vp]
    lib.gsvdec_attention_backward.argtypes = [_vp, ctypes.c_int, _vp]
    lib.gsvdec_ops_status.argtypes = [ctypes.c_int, _vp]
    lib.gsvdec_norm_workspace.argtypes = [_vp, sz]
    lib.gsvdec_norm_forward.argtypes = [_vp, ctypes.c_int, _vp]
    lib.gsvdec_norm_backward.argtypes = [_vp, ctypes.c_int, _vp]


class _Calls:
    """torch and the library's functions, looked up once."""

    def __init__(self):
        import torch
        from . import _check, library
        self.lib = lib = library()
        self.check = _check
        self.codes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        self.f32, self.i32, self.u8 = torch.float32, torch.int32, torch.uint8
        # Allocations are most of a small call's host time; these are the cheaper of torch's.
        self.empty_strided, self.empty_like = torch.empty_strided, torch.empty_like
        self.attention_forward, self.attention_backward = lib.gsvdec_attention_forward, lib.gsvdec_attention_backward
        self.norm_forward, self.norm_backward = lib.gsvdec_norm_forward, lib.gsvdec_norm_backward
        # The current stream's handle without building a torch Stream object, where torch offers that.
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        self.stream = raw or (lambda index: torch.cuda.current_stream(index).cuda_stream)


_calls = None


def _get() -> _Calls:
    global _calls
    if _calls is None:
        _calls = _Calls()
    return _calls


@functools.lru_cache(maxsize=4096)
def _attention_workspace(backward, dtype, B, H, Hkv, Tq, Tk, D, window, causal) -> int:
    a = _Attention()
    a.dtype, a.B, a.H, a.Hkv, a.Tq, a.Tk, a.D, a.window, a.causal = dtype, B, H, Hkv, Tq, Tk, D, window, causal
    a.scale = 1.0
    n, c = ctypes.c_size_t(), _get()
    c.check(c.lib.gsvdec_attention_workspace(ctypes.byref(a), backward, ctypes.byref(n)))
    return n.value


@functools.lru_cache(maxsize=4096)
def _norm_workspace(dtype, layout, B, C, T) -> int:
    a = _Norm()
    a.dtype, a.layout, a.B, a.C, a.T = dtype, layout, B, C, T
    n, c = ctypes.c_size_t(), _get()
    c.check(c.lib.gsvdec_norm_workspace(ctypes.byref(a), ctypes.byref(n)))
    return n.value


def _need(name, t, shape, dtype, index, contiguous=False) -> int:
    """Checks one tensor and returns its address."""
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, not {list(t.shape)}")
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, not on cuda:{index}")
    if contiguous:
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    elif t.stride(-1) != 1 and t.shape[-1] > 1 and t.numel():
        raise ValueError(f"{name}: the last axis must be contiguous")
    return t.data_ptr()


def _tensor(name, t, shape, dtype, index):
    """Checks one tensor; returns its address and strides (each of torch's accessors costs as much as the checks)."""
    s = t.stride()
    if t.shape == shape and t.dtype is dtype and t.get_device() == index and s[-1] == 1:
        return t.data_ptr(), s
    return _need(name, t, shape, dtype, index), s


def _first(name, t, ndim) -> int:
    if not t.is_cuda or t.dim() != ndim:
        raise ValueError(f"{name} must be a CUDA tensor with {ndim} axes")
    return t.get_device()


def _code(c, t) -> int:
    code = c.codes.get(t.dtype)
    if code is None:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, not {t.dtype}")
    return code


def _attention_in(c, q, k, v, scale, causal, q_lengths, k_lengths, rel_k, rel_v):
    """The checked inputs: (leading fields, addresses and strides up to rel_v, device index, strides of q, k, v)."""
    index = _first("q", q, 4)
    code, t = _code(c, q), q.dtype
    qs = q.shape
    B, H, Tq, D = qs
    if k.dim() != 4:
        raise ValueError("k must have 4 axes")
    ks = k.shape
    Hkv, Tk = ks[1], ks[2]
    if ks[0] != B or ks[3] != D:
        raise ValueError(f"k must be [{B}, heads, T, {D}], not {list(ks)}")
    pq, sq = _tensor("q", q, qs, t, index)
    pk, sk = _tensor("k", k, ks, t, index)
    pv, sv = _tensor("v", v, ks, t, index)
    ql = 0 if q_lengths is None else _need("q_lengths", q_lengths, (B,), c.i32, index, True)
    kl = 0 if k_lengths is None else _need("k_lengths", k_lengths, (B,), c.i32, index, True)
    window, rk, rv = -1, 0, 0
    if rel_k is not None or rel_v is not None:
        if rel_k is None or rel_v is None:
            raise ValueError("rel_k and rel_v come together")
        if rel_k.dim() != 2 or rel_k.shape[0] % 2 == 0:
            raise ValueError("rel_k must be [2 w + 1, D]")
        n = rel_k.shape[0]
        window = n // 2
        rk, rv = _need("rel_k", rel_k, (n, D), t, index, True), _need("rel_v", rel_v, (n, D), t, index, True)
    lead = (code, B, H, Hkv, Tq, Tk, D, window, 1 if causal else 0)
    if scale is None:
        scale = 1.0 / math.sqrt(D) if D else 1.0  # without channels: refused by the library
    given = (scale, ql, kl, pq, pk, pv, sq[0], sq[1], sq[2], sk[0], sk[1], sk[2], sv[0], sv[1], sv[2], rk, rv)
    return lead, given, index, (qs, ks, sq, sk, sv)


def _rows(c, dtype, n, m, device):
    """A new contiguous [n, m] tensor."""
    return c.empty_strided((n, m), (m, 1), dtype=dtype, device=device)


def _line(c, dtype, n, device):
    return c.empty_strided((n,), (1,), dtype=dtype, device=device)


def _same(c, x):
    """A new contiguous tensor of x's shape and type, and its leading strides."""
    _, m, n = x.shape
    t = c.empty_like(x) if x.is_contiguous() else c.empty_strided(x.shape, (m * n, n, 1), dtype=x.dtype, device=x.device)
    return t, m * n, n


def _heads_last(c, like, strides, B, H, T, D):
    """A new [B, H, T, D] tensor of like's type in [B, T, H, D] memory order, and its strides."""
    row = H * D
    s = (T * row, D, row, 1)
    if s == strides:  # like is in that order, and empty_like keeps it
        return c.empty_like(like), s
    return c.empty_strided((B, H, T, D), s, dtype=like.dtype, device=like.device), s


def attention(q, k, v, *, scale: Optional[float] = None, causal: bool = False, q_lengths=None, k_lengths=None,
              rel_k=None, rel_v=None):
    """softmax(scale q k^T + relative terms) v (MultiHeadAttention of the text
    encoder, src/models/sovits_encp.rs:98-102); returns (o, lse).

    q [B, H, Tq, D], k and v [B, Hkv, Tk, D] in fp32, fp16 or bf16 with any
    strides but a contiguous last axis; H a multiple of Hkv (query head h reads
    key head h / (H / Hkv)); D up to 128.  ``q_lengths`` / ``k_lengths`` [B]
    int32: valid rows.  The sequences are aligned at their ends: query i of
    utterance b stands at key position i + k_len - q_len, which ``causal`` and
    the offsets of ``rel_k`` / ``rel_v`` [2 w + 1, D] (learned relative keys and
    values, offsets -w .. w, w up to 15) count from.  Rows without an allowed
    key give o = 0 and lse = -inf.  o [B, H, Tq, D] has [B, Tq, H, D] memory
    order; lse [B, H, Tq] fp32 is the log-sum-exp of each row's scores.
    """
    c = _get()
    lead, given, index, (_, _, sq, _, _) = _attention_in(c, q, k, v, scale, causal, q_lengths, k_lengths, rel_k, rel_v)
    code, B, H, _, Tq, _, D = lead[:7]
    dev = q.device
    o, so = _heads_last(c, q, sq, B, H, Tq, D)
    lse = c.empty_strided((B, H, Tq), (H * Tq, Tq, 1), dtype=c.f32, device=dev)
    n = _attention_workspace(0, *lead)
    ws = _line(c, c.u8, n, dev) if n else None
    a = _ATTENTION.pack(*lead, *given, o.data_ptr(), *so[:3], lse.data_ptr(), 0, *_Z3, 0, 0, 0, *_Z3, *_Z3, *_Z3, 0, 0,
                        ws.data_ptr() if n else 0, n)
    rc = c.attention_forward(a, index, c.stream(index))
    if rc:
        c.check(rc)
    return o, lse


def attention_backward(do, q, k, v, o, lse, *, scale: Optional[float] = None, causal: bool = False, q_lengths=None,
                       k_lengths=None, rel_k=None, rel_v=None):
    """Gradients (dq, dk, dv, drel_k, drel_v) of :func:`attention` for the
    gradient ``do`` of its first result; ``o`` and ``lse`` are its results and
    the other arguments those it was called with.  The probabilities are
    recomputed from lse.  drel_k and drel_v are None without a window; every
    gradient has its input's type (gradients of shared key heads and of the
    relative rows are summed in fp32 and rounded once) and is bit-reproducible.
    """
    c = _get()
    lead, given, index, (qs, _, sq, sk, sv) = _attention_in(c, q, k, v, scale, causal, q_lengths, k_lengths, rel_k,
                                                            rel_v)
    code, B, H, Hkv, Tq, Tk, D, window = lead[:8]
    t = q.dtype
    pdo, sdo = _tensor("do", do, qs, t, index)
    po, so = _tensor("o", o, qs, t, index)
    pl = _need("lse", lse, (B, H, Tq), c.f32, index, True)
    dev = q.device
    dq, sq = _heads_last(c, q, sq, B, H, Tq, D)
    dk, sk = _heads_last(c, k, sk, B, Hkv, Tk, D)
    dv, sv = _heads_last(c, v, sv, B, Hkv, Tk, D)
    drk = drv = None
    prk = prv = 0
    if window >= 0:
        drk, drv = c.empty_like(rel_k), c.empty_like(rel_v)
        prk, prv = drk.data_ptr(), drv.data_ptr()
    n = _attention_workspace(1, *lead)
    ws = _line(c, c.u8, n, dev)
    a = _ATTENTION.pack(*lead, *given, po, *so[:3], pl, pdo, *sdo[:3], dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                        *sq[:3], *sk[:3], *sv[:3], prk, prv, ws.data_ptr(), n)
    rc = c.attention_backward(a, index, c.stream(index))
    if rc:
        c.check(rc)
    return dq, dk, dv, drk, drv


def _index(device) -> int:
    import torch
    index = None if device is None else torch.device(device).index
    return torch.cuda.current_device() if index is None else index


def ops_status(device=None) -> None:
    """Waits for the current stream of ``device`` (default: the current one) and
    raises GsvDecError(GSV_E_TIMEOUT) if a bounded device wait of an operator
    there gave up since this thread's last call (gsvdec_ops_status)."""
    index, c = _index(device), _get()
    c.check(c.lib.gsvdec_ops_status(index, c.stream(index)))


def selftest_wait(limit_ns: int = 1_000_000, device=None) -> None:
    """Queue a bounded wait that nothing completes on the current stream of
    ``device``; ops_status then reports it like an operator's give-up
    (gsvdec_selftest_attention_wait)."""
    index, c = _index(device), _get()
    c.check(c.lib.gsvdec_selftest_attention_wait(None, index, int(limit_ns), c.stream(index)))


def _norm_in(c, x, y, lengths, layout):
    index = _first("x", x, 3)
    code, t, xs = _code(c, x), x.dtype, x.shape
    lay = LAYOUTS.get(layout)
    if lay is None:
        raise ValueError(f"layout must be one of {sorted(LAYOUTS)}")
    B, C, T = xs if lay == 0 else (xs[0], xs[2], xs[1])
    px, sx = _tensor("x", x, xs, t, index)
    py, sy = (0, (0, 0)) if y is None else _tensor("y", y, xs, t, index)
    ln = 0 if lengths is None else _need("lengths", lengths, (B,), c.i32, index, True)
    return (code, lay, B, C, T), (ln, px, py, sx[0], sx[1], sy[0], sy[1]), index


def add_norm(x, y, gamma, beta, *, lengths=None, layout: str = "bct", eps: float = 1e-5):
    """LayerNorm over channels of x + y (norm1(x + attn(x)) of
    EncoderLayer::forward, src/models/sovits_encp.rs:102); returns (out, mean,
    rstd).

    x, y (or None) [B, C, T] (layout "bct", C up to 2048) or [B, T, C] ("btc",
    C up to 8192) in fp32, fp16 or bf16; gamma, beta [C] fp32; lengths [B]
    int32.  mean and rstd [B, T] fp32 are what :func:`add_norm_backward` needs.
    Frames t >= lengths[b] give out = mean = rstd = 0.
    """
    c = _get()
    lead, given, index = _norm_in(c, x, y, lengths, layout)
    B, C, T = lead[2:]
    pg, pb = _need("gamma", gamma, (C,), c.f32, index, True), _need("beta", beta, (C,), c.f32, index, True)
    dev = x.device
    out, s0, s1 = _same(c, x)
    mean = _rows(c, c.f32, B, T, dev)
    rstd = c.empty_like(mean)
    a = _NORM.pack(*lead, eps, *given, pg, pb, mean.data_ptr(), rstd.data_ptr(), out.data_ptr(), s0, s1, 0, 0,
                   0, 0, 0, 0, 0, 0, 0, 0)
    rc = c.norm_forward(a, index, c.stream(index))
    if rc:
        c.check(rc)
    return out, mean, rstd


def add_norm_backward(d_out, x, y, gamma, mean, rstd, *, lengths=None, layout: str = "bct"):
    """Gradients (dx, dgamma, dbeta) of :func:`add_norm`; dx is the gradient of
    x and of y.  mean and rstd are add_norm's.  dgamma and dbeta are fp32 sums
    over the frames in a fixed order."""
    c = _get()
    lead, given, index = _norm_in(c, x, y, lengths, layout)
    B, C, T = lead[2:]
    pg = _need("gamma", gamma, (C,), c.f32, index, True)
    pd, sd = _tensor("d_out", d_out, x.shape, x.dtype, index)
    pm, pr = _need("mean", mean, (B, T), c.f32, index, True), _need("rstd", rstd, (B, T), c.f32, index, True)
    dev = x.device
    dx, s0, s1 = _same(c, x)
    dgamma, dbeta = c.empty_like(gamma), c.empty_like(gamma)
    n = _norm_workspace(*lead)
    ws = _line(c, c.u8, n, dev)
    a = _NORM.pack(*lead, 0.0, *given, pg, 0, pm, pr, 0, 0, 0, pd, dx.data_ptr(), sd[0], sd[1],
                   s0, s1, dgamma.data_ptr(), dbeta.data_ptr(), ws.data_ptr(), n)
    rc = c.norm_backward(a, index, c.stream(index))
    if rc:
        c.check(rc)
    return dx, dgamma, dbeta
