"""Operators on tensors whose elements lie further than 2^32 elements apart (a
long cache): rows of every tensor, outputs included, are strided over one large
buffer.  The results have to be those of the same call on contiguous tensors, bit
for bit: both move by the same kernels."""
from __future__ import annotations

import ctypes

import pytest
import torch

from attn_ref import TYPES

pytestmark = pytest.mark.gpu

T = 300
STEP = ((1 << 32) // (T - 1) + 4096) // 64 * 64  # the last row lies past 2^32 elements
ROOM = T * STEP


@pytest.fixture(scope="module", params=["bf16", "fp16", "fp32"])
def buffer(request):
    t = TYPES[request.param]
    if torch.cuda.mem_get_info()[0] < ROOM * t.itemsize + (4 << 30):
        pytest.skip("needs 17 GB of device memory")
    b = torch.empty(ROOM, dtype=t, device="cuda")
    yield b
    del b
    torch.cuda.empty_cache()


class Places:
    """Tensors whose axis `far` steps by STEP, the others inside a step."""

    def __init__(self, buf):
        self.buf, self.at = buf, 0

    def __call__(self, shape, far):
        s, near = [0] * len(shape), 1
        for i in reversed(range(len(shape))):
            if i == far:
                s[i] = STEP
            else:
                s[i] = near
                near *= shape[i]
        t = torch.as_strided(self.buf, shape, s, self.at)
        self.at += (near + 63) // 64 * 64
        assert self.at <= STEP and shape[far] <= T
        return t

    def copy(self, x, far):
        t = self(tuple(x.shape), far)
        t.copy_(x)
        return t


def run(f, a):
    from torch.cuda import current_stream
    assert f(ctypes.byref(a), 0, ctypes.c_void_p(current_stream().cuda_stream)) == 0


@pytest.mark.parametrize("Tq,H,Hkv,D,w", [(T, 2, 2, 64, 4), (T, 4, 2, 96, -1), (2, 4, 2, 64, 3), (1, 2, 1, 128, -1)])
def test_attention(gsv, buffer, Tq, H, Hkv, D, w):
    t = buffer.dtype
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda n, h: torch.randn(2, h, n, D, generator=g, device="cuda").to(t)  # noqa: E731
    q, k, v, do = r(Tq, H), r(T, Hkv), r(T, Hkv), r(Tq, H)
    n = torch.tensor([T, T - 7], dtype=torch.int32, device="cuda")
    rel = {} if w < 0 else {x: (torch.randn(2 * w + 1, D, generator=g, device="cuda") * 0.1).to(t)
                            for x in ("rel_k", "rel_v")}
    kw = dict(k_lengths=n, causal=True, **rel)
    o, lse = gsv.attention(q, k, v, **kw)
    grads = gsv.attention_backward(do, q, k, v, o, lse, **kw)
    p = Places(buffer)
    far = {"q": p.copy(q, 2), "k": p.copy(k, 2), "v": p.copy(v, 2), "d_o": p.copy(do, 2)}
    # Through the Python call: inputs far apart.
    o2, lse2 = gsv.attention(far["q"], far["k"], far["v"], **kw)
    assert torch.equal(o2, o) and torch.equal(lse2, lse)
    for a, b in zip(gsv.attention_backward(far["d_o"], far["q"], far["k"], far["v"], o2, lse2, **kw), grads):
        assert (a is None and b is None) or torch.equal(a, b)
    # Through the C call: outputs too.
    far.update(o=p(tuple(o.shape), 2), dq=p(tuple(q.shape), 2), dk=p(tuple(k.shape), 2), dv=p(tuple(k.shape), 2))
    a = gsv.ops._Attention()
    a.dtype, a.B, a.H, a.Hkv, a.Tq, a.Tk, a.D, a.window, a.causal = gsv.ops._get().codes[t], 2, H, Hkv, Tq, T, D, w, 1
    a.scale = D ** -0.5
    for name, x in far.items():
        setattr(a, name, x.data_ptr())
        getattr(a, name + "_stride")[:] = x.stride()[:3]
    lse3, drel = torch.empty_like(lse), {x: torch.empty_like(y) for x, y in rel.items()}
    a.lse, a.k_lengths = lse3.data_ptr(), n.data_ptr()
    for x, y in rel.items():
        setattr(a, x, y.data_ptr())
        setattr(a, "d" + x, drel[x].data_ptr())
    size = gsv.ops._attention_workspace(1, a.dtype, 2, H, Hkv, Tq, T, D, w, 1)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), size
    lib = gsv.library()
    run(lib.gsvdec_attention_forward, a)
    run(lib.gsvdec_attention_backward, a)
    assert torch.equal(far["o"], o) and torch.equal(lse3, lse)
    for x, want in zip(("dq", "dk", "dv"), grads):
        assert torch.equal(far[x], want), x
    for x, want in zip(("rel_k", "rel_v"), grads[3:]):
        assert want is None or torch.equal(drel[x], want)
    gsv.ops_status()


@pytest.mark.parametrize("layout,shape", [("btc", (2, T, 192)), ("btc", (3, T, 515)), ("bct", (2, T, 44)),
                                          ("bct", (2, T, 45))])
def test_norm(gsv, buffer, layout, shape):
    t = buffer.dtype
    g = torch.Generator(device="cuda").manual_seed(2)
    x, y, d_out = (torch.randn(shape, generator=g, device="cuda").to(t) for _ in range(3))
    C = shape[1] if layout == "bct" else shape[2]
    gamma, beta = (torch.randn(C, generator=g, device="cuda") for _ in range(2))
    out, mean, rstd = gsv.add_norm(x, y, gamma, beta, layout=layout)
    dx, dgamma, dbeta = gsv.add_norm_backward(d_out, x, y, gamma, mean, rstd, layout=layout)
    p = Places(buffer)
    far = {"x": p.copy(x, 1), "y": p.copy(y, 1), "d_out": p.copy(d_out, 1), "out": p(shape, 1), "dx": p(shape, 1)}
    a = gsv.ops._Norm()
    a.dtype, a.layout, a.B, a.C, a.T = gsv.ops._get().codes[t], gsv.ops.LAYOUTS[layout], shape[0], C, \
        shape[2] if layout == "bct" else shape[1]
    a.eps = 1e-5
    for name, z in far.items():
        setattr(a, name, z.data_ptr())
        getattr(a, name + "_stride")[:] = z.stride()[:2]
    kept = {"gamma": gamma, "beta": beta, "mean": torch.empty_like(mean), "rstd": torch.empty_like(rstd),
            "dgamma": torch.empty_like(gamma), "dbeta": torch.empty_like(gamma)}
    for name, z in kept.items():
        setattr(a, name, z.data_ptr())
    size = gsv.ops._norm_workspace(a.dtype, a.layout, a.B, a.C, a.T)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), size
    lib = gsv.library()
    run(lib.gsvdec_norm_forward, a)
    run(lib.gsvdec_norm_backward, a)
    for name, want in (("out", out), ("dx", dx)):
        assert torch.equal(far[name], want), name
    for name, want in (("mean", mean), ("rstd", rstd), ("dgamma", dgamma), ("dbeta", dbeta)):
        assert torch.equal(kept[name], want), name
    gsv.ops_status()
