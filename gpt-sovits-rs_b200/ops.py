"""Attention and residual norm of the text encoder with their gradients, on CUDA tensors.

Stand-alone operators over ``gsvdec_attention_*`` and ``gsvdec_norm_*``
(include/gsvdec.h): no handle and no state.  Each call runs on the current
stream of its tensors' device, takes outputs and workspace from torch's
allocator, does not synchronise and can be captured in a CUDA graph.  The
forward calls return what their backward needs.
"""
from __future__ import annotations

import ctypes
import math
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


def declare(lib) -> None:
    """Argument types of the operators' C functions."""
    at, nt, sz = ctypes.POINTER(_Attention), ctypes.POINTER(_Norm), ctypes.POINTER(ctypes.c_size_t)
    lib.gsvdec_attention_workspace.argtypes = [at, ctypes.c_int, sz]
    lib.gsvdec_attention_forward.argtypes = [at, ctypes.c_int, _vp]
    lib.gsvdec_attention_backward.argtypes = [at, ctypes.c_int, _vp]
    lib.gsvdec_ops_status.argtypes = [ctypes.c_int, _vp]
    lib.gsvdec_norm_workspace.argtypes = [nt, sz]
    lib.gsvdec_norm_forward.argtypes = [nt, ctypes.c_int, _vp]
    lib.gsvdec_norm_backward.argtypes = [nt, ctypes.c_int, _vp]


def _lib():
    from . import library
    return library()


def _check(rc: int) -> None:
    if rc:
        from . import _check as check
        check(rc)


def _dtype(t) -> int:
    import torch
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}.get(t.dtype)
    if code is None:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, not {t.dtype}")
    return code


def _take(name, t, shape, dtype, device, contiguous=False):
    """Checks one tensor and returns its address (None stays None)."""
    if t is None:
        return None
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, not {list(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if not contiguous and t.shape[-1] > 1 and t.stride(-1) != 1 and t.numel():
        raise ValueError(f"{name}: the last axis must be contiguous")
    return t.data_ptr()


def _run(call, a, device) -> None:
    import torch
    _check(call(ctypes.byref(a), device.index, torch.cuda.current_stream(device).cuda_stream))


def _cuda(name, t, ndim):
    if not t.is_cuda or t.dim() != ndim:
        raise ValueError(f"{name} must be a CUDA tensor with {ndim} axes")
    return t.device


def _attention_args(q, k, v, scale, causal, q_lengths, k_lengths, rel_k, rel_v):
    import torch
    dev = _cuda("q", q, 4)
    if k.dim() != 4:
        raise ValueError("k must have 4 axes")
    B, H, Tq, D = q.shape
    Hkv, Tk = k.shape[1], k.shape[2]
    a = _Attention()
    a.dtype = _dtype(q)
    a.B, a.H, a.Hkv, a.Tq, a.Tk, a.D = B, H, Hkv, Tq, Tk, D
    a.causal = 1 if causal else 0
    a.scale = 1.0 / math.sqrt(D) if scale is None else scale
    a.q = _take("q", q, (B, H, Tq, D), q.dtype, dev)
    a.k = _take("k", k, (B, Hkv, Tk, D), q.dtype, dev)
    a.v = _take("v", v, (B, Hkv, Tk, D), q.dtype, dev)
    a.q_stride[:], a.k_stride[:], a.v_stride[:] = q.stride()[:3], k.stride()[:3], v.stride()[:3]
    a.q_lengths = _take("q_lengths", q_lengths, (B,), torch.int32, dev, True)
    a.k_lengths = _take("k_lengths", k_lengths, (B,), torch.int32, dev, True)
    if (rel_k is None) != (rel_v is None):
        raise ValueError("rel_k and rel_v come together")
    a.window = -1
    if rel_k is not None:
        n = rel_k.shape[0]
        if rel_k.dim() != 2 or n % 2 == 0:
            raise ValueError("rel_k must be [2 w + 1, D]")
        a.window = n // 2
        a.rel_k = _take("rel_k", rel_k, (n, D), q.dtype, dev, True)
        a.rel_v = _take("rel_v", rel_v, (n, D), q.dtype, dev, True)
    return a, dev


def _workspace(a, backward, dev):
    import torch
    n = ctypes.c_size_t()
    _check(_lib().gsvdec_attention_workspace(ctypes.byref(a), backward, ctypes.byref(n)))
    ws = None
    if n.value:
        ws = torch.empty(n.value, dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = ws.data_ptr(), n.value
    return ws


def _like(t):
    """A new tensor of t's shape in [B, T, heads, D] memory order."""
    import torch
    B, H, T, D = t.shape
    return torch.empty((B, T, H, D), dtype=t.dtype, device=t.device).transpose(1, 2)


def attention(q, k, v, *, scale: Optional[float] = None, causal: bool = False, q_lengths=None, k_lengths=None,
              rel_k=None, rel_v=None):
    """softmax(scale q k^T + relative terms) v (MultiHeadAttention of the text
    encoder, src/models/sovits_encp.rs:98-102); returns (o, lse).

    q [B, H, Tq, D], k and v [B, Hkv, Tk, D] in fp32, fp16 or bf16 with any
    strides but a contiguous last axis; H a multiple of Hkv (query head h reads
    key head h / (H / Hkv)).  ``q_lengths`` / ``k_lengths`` [B] int32: valid
    rows.  The sequences are aligned at their ends: query i of utterance b
    stands at key position i + k_len - q_len, which ``causal`` and the offsets
    of ``rel_k`` / ``rel_v`` [2 w + 1, D] (learned relative keys and values,
    offsets -w .. w) count from.  Rows without an allowed key give o = 0 and
    lse = -inf.  o [B, H, Tq, D] has [B, Tq, H, D] memory order; lse
    [B, H, Tq] fp32 is the log-sum-exp of each row's scores.
    """
    import torch
    a, dev = _attention_args(q, k, v, scale, causal, q_lengths, k_lengths, rel_k, rel_v)
    o = _like(q)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=dev)
    a.o, a.lse = o.data_ptr(), lse.data_ptr()
    a.o_stride[:] = o.stride()[:3]
    ws = _workspace(a, 0, dev)  # noqa: F841  (alive until the call has queued its kernels)
    _run(_lib().gsvdec_attention_forward, a, dev)
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
    import torch
    a, dev = _attention_args(q, k, v, scale, causal, q_lengths, k_lengths, rel_k, rel_v)
    a.d_o = _take("do", do, tuple(q.shape), q.dtype, dev)
    a.o = _take("o", o, tuple(q.shape), q.dtype, dev)
    a.lse = _take("lse", lse, tuple(q.shape[:3]), torch.float32, dev, True)
    a.d_o_stride[:], a.o_stride[:] = do.stride()[:3], o.stride()[:3]
    dq, dk, dv = _like(q), _like(k), _like(k)
    a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    a.dq_stride[:], a.dk_stride[:], a.dv_stride[:] = dq.stride()[:3], dk.stride()[:3], dv.stride()[:3]
    drk = drv = None
    if rel_k is not None:
        drk, drv = torch.empty_like(rel_k), torch.empty_like(rel_v)
        a.drel_k, a.drel_v = drk.data_ptr(), drv.data_ptr()
    ws = _workspace(a, 1, dev)  # noqa: F841
    _run(_lib().gsvdec_attention_backward, a, dev)
    return dq, dk, dv, drk, drv


def ops_status(device=None) -> None:
    """Waits for the current stream of ``device`` (default: the current one) and
    raises GsvDecError(GSV_E_TIMEOUT) if a bounded device wait of an operator
    there gave up (gsvdec_ops_status)."""
    import torch
    index = torch.cuda.current_device() if device is None else torch.device(device).index
    _check(_lib().gsvdec_ops_status(index, torch.cuda.current_stream(index).cuda_stream))


def _norm_args(x, y, gamma, beta, lengths, layout, eps):
    import torch
    dev = _cuda("x", x, 3)
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {sorted(LAYOUTS)}")
    a = _Norm()
    a.dtype, a.layout = _dtype(x), LAYOUTS[layout]
    a.B = x.shape[0]
    a.C, a.T = (x.shape[1], x.shape[2]) if layout == "bct" else (x.shape[2], x.shape[1])
    a.eps = eps
    a.x = _take("x", x, tuple(x.shape), x.dtype, dev)
    a.y = _take("y", y, tuple(x.shape), x.dtype, dev)
    a.x_stride[:] = x.stride()[:2]
    if y is not None:
        a.y_stride[:] = y.stride()[:2]
    a.gamma = _take("gamma", gamma, (a.C,), torch.float32, dev, True)
    a.beta = _take("beta", beta, (a.C,), torch.float32, dev, True)
    a.lengths = _take("lengths", lengths, (a.B,), torch.int32, dev, True)
    return a, dev


def add_norm(x, y, gamma, beta, *, lengths=None, layout: str = "bct", eps: float = 1e-5):
    """LayerNorm over channels of x + y (norm1(x + attn(x)) of
    EncoderLayer::forward, src/models/sovits_encp.rs:102); returns (out, mean,
    rstd).

    x, y (or None) [B, C, T] (layout "bct") or [B, T, C] ("btc") in fp32, fp16
    or bf16; gamma, beta [C] fp32; lengths [B] int32.  mean and rstd [B, T]
    fp32 are what :func:`add_norm_backward` needs.  Frames t >= lengths[b] give
    out = mean = rstd = 0.
    """
    import torch
    a, dev = _norm_args(x, y, gamma, beta, lengths, layout, eps)
    out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    mean, rstd = torch.empty((2, a.B, a.T), dtype=torch.float32, device=dev).unbind(0)
    a.out, a.mean, a.rstd = out.data_ptr(), mean.data_ptr(), rstd.data_ptr()
    a.out_stride[:] = out.stride()[:2]
    _run(_lib().gsvdec_norm_forward, a, dev)
    return out, mean, rstd


def add_norm_backward(d_out, x, y, gamma, mean, rstd, *, lengths=None, layout: str = "bct"):
    """Gradients (dx, dgamma, dbeta) of :func:`add_norm`; dx is the gradient of
    x and of y.  mean and rstd are add_norm's.  dgamma and dbeta are fp32 sums
    over the frames in a fixed order."""
    import torch
    a, dev = _norm_args(x, y, gamma, None, lengths, layout, 0.0)
    a.d_out = _take("d_out", d_out, tuple(x.shape), x.dtype, dev)
    a.d_out_stride[:] = d_out.stride()[:2]
    a.mean = _take("mean", mean, (a.B, a.T), torch.float32, dev, True)
    a.rstd = _take("rstd", rstd, (a.B, a.T), torch.float32, dev, True)
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
    dgamma, dbeta = torch.empty((2, a.C), dtype=torch.float32, device=dev).unbind(0)
    a.dx, a.dgamma, a.dbeta = dx.data_ptr(), dgamma.data_ptr(), dbeta.data_ptr()
    a.dx_stride[:] = dx.stride()[:2]
    n = ctypes.c_size_t()
    _check(_lib().gsvdec_norm_workspace(ctypes.byref(a), ctypes.byref(n)))
    ws = torch.empty(n.value, dtype=torch.uint8, device=dev)
    a.workspace, a.workspace_bytes = ws.data_ptr(), n.value
    _run(_lib().gsvdec_norm_backward, a, dev)
    return dx, dgamma, dbeta
