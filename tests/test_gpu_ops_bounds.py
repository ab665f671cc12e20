"""What the operators write: every element of their outputs and nothing beside
them, in tensors that are slices of larger ones, with guards behind the
workspace and the statistics."""
from __future__ import annotations

import ctypes

import pytest
import torch

import test_gpu_norm as norm
from attn_ref import TYPES, check, reference

pytestmark = pytest.mark.gpu

MARK = 77.0


class Guarded:
    """Slices of marked buffers; untouched() says whether the rest of them is still marked."""

    def __init__(self):
        self.kept = []

    def slice(self, shape, dtype, pads):
        big = torch.full([n + p[0] + p[1] for n, p in zip(shape, pads)], MARK, dtype=dtype, device="cuda")
        view = big[tuple(slice(p[0], p[0] + n) for n, p in zip(shape, pads))]
        self.kept.append((big, view))
        return view

    def flat(self, n, dtype):
        return self.slice((n,), dtype, [(64, 64)])  # the front part keeps the alignment

    def untouched(self):
        ok = True
        for big, view in self.kept:
            rest = big.clone()
            torch.as_strided(rest, view.shape, view.stride(), view.storage_offset()).fill_(MARK)
            ok = ok and bool((rest == MARK).all())
        return ok

    def written(self):
        return all(bool((view != MARK).any()) or view.numel() == 0 for _, view in self.kept)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("D,pad", [(20, 3), (24, 8), (33, 1), (64, 16), (80, 16), (96, 8), (128, 32)])
@pytest.mark.parametrize("Tq,Tk,w", [(131, 70, 4), (70, 1100, -1), (2, 300, 2), (64, 64, 15)])
def test_attention(gsv, dtype, D, pad, Tq, Tk, w):
    t = TYPES[dtype]
    B, H, Hkv = 2, 2, 1
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda n, h: torch.randn(B, n, h, D, generator=g, device="cuda").to(t).transpose(1, 2)  # noqa: E731
    q, k, v, do = r(Tq, H), r(Tk, Hkv), r(Tk, Hkv), r(Tq, H)
    ql, kl = (torch.tensor(n, dtype=torch.int32, device="cuda") for n in ((Tq, Tq // 2), (Tk - 3, Tk // 3)))
    rel = {} if w < 0 else {x: (torch.randn(2 * w + 1, D, generator=g, device="cuda") * 0.1).to(t)
                            for x in ("rel_k", "rel_v")}
    out = Guarded()
    rows = lambda n, h: out.slice((B, n, h, D), t, [(0, 0), (1, 2), (0, 0), (pad, pad)]).transpose(1, 2)  # noqa: E731
    a = gsv.ops._Attention()
    a.dtype, a.B, a.H, a.Hkv, a.Tq, a.Tk, a.D, a.window, a.causal = gsv.ops._get().codes[t], B, H, Hkv, Tq, Tk, D, w, 1
    a.scale = D ** -0.5
    x = {"q": q, "k": k, "v": v, "d_o": do, "o": rows(Tq, H), "dq": rows(Tq, H), "dk": rows(Tk, Hkv), "dv": rows(Tk, Hkv)}
    for name, z in x.items():
        setattr(a, name, z.data_ptr())
        getattr(a, name + "_stride")[:] = z.stride()[:3]
    lse2 = out.flat(B * H * Tq, torch.float32)
    drel = {n: out.flat(y.numel(), t) for n, y in rel.items()}
    a.lse, a.q_lengths, a.k_lengths = lse2.data_ptr(), ql.data_ptr(), kl.data_ptr()
    for n, y in rel.items():
        setattr(a, n, y.data_ptr())
        setattr(a, "d" + n, drel[n].data_ptr())
    size = gsv.ops._attention_workspace(1, a.dtype, B, H, Hkv, Tq, Tk, D, w, 1)
    ws = Guarded()
    a.workspace, a.workspace_bytes = ws.flat(size // 4, torch.float32).data_ptr(), size
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert gsv.library().gsvdec_attention_forward(ctypes.byref(a), 0, st) == 0
    assert gsv.library().gsvdec_attention_backward(ctypes.byref(a), 0, st) == 0
    assert out.untouched() and out.written() and ws.untouched()
    ref = reference(q, k, v, do, q_lengths=ql, k_lengths=kl, causal=True, **rel)
    for name in ("o", "dq", "dk", "dv"):
        check(name, x[name], ref, t)
    check("lse", lse2.view(B, H, Tq), ref, torch.float32)
    for n, z in drel.items():
        check("d" + n, z.view(-1, D), ref, t)
    gsv.ops_status()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("layout,C,T", [("btc", 192, 50), ("btc", 515, 33), ("btc", 1024, 40), ("bct", 192, 50),
                                        ("bct", 700, 33), ("bct", 5, 64)])
@pytest.mark.parametrize("pad", [1, 8])
def test_norm(gsv, dtype, layout, C, T, pad):
    t, B = TYPES[dtype], 3
    g = torch.Generator(device="cuda").manual_seed(0)
    shape = (B, T, C) if layout == "btc" else (B, C, T)
    x, y, d_out = (torch.randn(shape, generator=g, device="cuda").to(t) for _ in range(3))
    gamma, beta = (torch.randn(C, generator=g, device="cuda") for _ in range(2))
    n = torch.tensor([T, 0, T // 2], dtype=torch.int32, device="cuda")
    ref = norm.reference({"x": x, "y": y, "d_out": d_out, "gamma": gamma, "beta": beta}, layout, n)
    out = Guarded()
    a = gsv.ops._Norm()
    a.dtype, a.layout, a.B, a.C, a.T = gsv.ops._get().codes[t], gsv.ops.LAYOUTS[layout], B, C, T
    a.eps = 1e-5
    z = {"x": x, "y": y, "d_out": d_out}
    for name in ("out", "dx"):
        z[name] = out.slice(shape, t, [(0, 0), (1, 1), (pad, pad)])
    for name, s in z.items():
        setattr(a, name, s.data_ptr())
        getattr(a, name + "_stride")[:] = s.stride()[:2]
    kept = {"gamma": gamma, "beta": beta}
    for name, m in (("mean", B * T), ("rstd", B * T), ("dgamma", C), ("dbeta", C)):
        kept[name] = out.flat(m, torch.float32)
    for name, s in kept.items():
        setattr(a, name, s.data_ptr())
    size = gsv.ops._norm_workspace(a.dtype, a.layout, B, C, T)
    ws = Guarded()
    a.workspace, a.workspace_bytes, a.lengths = ws.flat(size // 4, torch.float32).data_ptr(), size, n.data_ptr()
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert gsv.library().gsvdec_norm_forward(ctypes.byref(a), 0, st) == 0
    assert gsv.library().gsvdec_norm_backward(ctypes.byref(a), 0, st) == 0
    assert out.untouched() and out.written() and ws.untouched()
    for name in ("out", "dx"):
        norm.check(name, z[name], ref, t)
    for name in ("mean", "rstd"):
        norm.check(name, kept[name].view(B, T), ref)
    for name in ("dgamma", "dbeta"):
        norm.check(name, kept[name], ref)
    gsv.ops_status()
