"""The operators as a training step uses them: the attention half of an encoder
layer (projections, attention with relative keys and values, output projection,
residual norm) under torch autograd, against autograd of the plain formulas in
64 bits.

Tolerance: each of the three stages is a chain of fp32 sums over at most
192 + 100 terms, off by 2 (n + 64) 2^-24 of its terms' absolute sum, which for
these random inputs stays within twice the result's largest value: 3 stages x
2 x 2 x 356 x 6e-8 = 2.6e-4 of the largest value of each result."""
from __future__ import annotations

import pytest
import torch

from attn_ref import geometry

pytestmark = pytest.mark.gpu

TOL = 2.6e-4
C, H, W = 192, 2, 4
D = C // H


def functions(gsv):
    class Attention(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v, rel_k, rel_v, lengths):
            kw = dict(q_lengths=lengths, k_lengths=lengths, rel_k=rel_k, rel_v=rel_v)
            o, lse = gsv.attention(q, k, v, **kw)
            ctx.save_for_backward(q, k, v, o, lse, rel_k, rel_v, lengths)
            return o

        @staticmethod
        def backward(ctx, do):
            q, k, v, o, lse, rel_k, rel_v, n = ctx.saved_tensors
            return gsv.attention_backward(do, q, k, v, o, lse, q_lengths=n, k_lengths=n, rel_k=rel_k, rel_v=rel_v) \
                + (None,)

    class AddNorm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, y, gamma, beta, lengths):
            out, mean, rstd = gsv.add_norm(x, y, gamma, beta, lengths=lengths, layout="btc")
            ctx.save_for_backward(x, y, gamma, mean, rstd, lengths)
            return out

        @staticmethod
        def backward(ctx, d_out):
            x, y, gamma, mean, rstd, n = ctx.saved_tensors
            dx, dg, db = gsv.add_norm_backward(d_out.contiguous(), x, y, gamma, mean, rstd, lengths=n, layout="btc")
            return dx, dx, dg, db, None

    return Attention.apply, AddNorm.apply


def parameters(dtype):
    g = torch.Generator().manual_seed(0)
    r = lambda *s, std=1.0: (torch.randn(s, generator=g) * std).to("cuda", dtype).requires_grad_()  # noqa: E731
    p = {n: r(C, C, std=C ** -0.5) for n in ("wq", "wk", "wv", "wo")}
    p.update(rel_k=r(2 * W + 1, D, std=D ** -0.5), rel_v=r(2 * W + 1, D, std=D ** -0.5), gamma=r(C), beta=r(C))
    return p


def heads(x, w):
    B, T, _ = x.shape
    return (x @ w.T).view(B, T, H, D).transpose(1, 2)


def plain_attention(q, k, v, rel_k, rel_v, n):
    B, _, T, _ = q.shape
    ok, r = geometry(B, T, T, n, n, False, q.device)
    near, idx = (r.abs() <= W) & ok, (r + W).clamp(0, 2 * W)
    idx = idx.expand(B, H, T, T)
    s = q @ k.transpose(-1, -2) + torch.where(near, (q @ rel_k.T).gather(-1, idx), 0.0)
    p = torch.softmax((s * D ** -0.5).masked_fill(~ok, -1e30), -1) * ok
    o = p @ v
    for j in range(-W, W + 1):
        o = o + (p * (near & (r == j))).sum(-1, keepdim=True) * rel_v[j + W]
    return o


def plain_norm(x, y, gamma, beta, n):
    s = x + y
    s = (s - s.mean(-1, keepdim=True)) / torch.sqrt(s.var(-1, unbiased=False, keepdim=True) + 1e-5) * gamma + beta
    ok = torch.arange(x.shape[1], device=x.device).view(1, -1, 1) < n.view(-1, 1, 1)
    return s * ok


def step(x, p, n, weight, attention, norm):
    o = attention(heads(x, p["wq"]), heads(x, p["wk"]), heads(x, p["wv"]), p["rel_k"], p["rel_v"], n)
    y = o.transpose(1, 2).reshape(x.shape) @ p["wo"].T
    out = norm(x, y, p["gamma"], p["beta"], n)
    (out * weight).sum().backward()
    return out


def test_one_training_step(gsv):
    B, T = 3, 100
    n = torch.tensor([100, 61, 8], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(1)
    x0, w0 = torch.randn(B, T, C, generator=g).cuda(), torch.randn(B, T, C, generator=g).cuda()
    results = []
    for dtype, fns in ((torch.float32, functions(gsv)), (torch.float64, (plain_attention, plain_norm))):
        p = parameters(torch.float32)
        p = {k: v.detach().to(dtype).requires_grad_() for k, v in p.items()}
        x = x0.to(dtype, copy=True).requires_grad_()
        out = step(x, p, n, w0.to(dtype), *fns)
        results.append({"out": out.detach(), "x": x.grad, **{k: v.grad for k, v in p.items()}})
    for name, want in results[1].items():
        got = results[0][name].double()
        off = (got - want).abs().max() / want.abs().max()
        assert off <= TOL, f"{name}: {off:.2e}"


def test_half_precision_step_runs_and_repeats(gsv):
    # The same step in bf16: it runs, its gradients are finite, and a second pass gives the same bits.
    attention, norm = functions(gsv)
    n = torch.tensor([64, 40], dtype=torch.int32, device="cuda")
    first = None
    for _ in range(2):
        p = {k: (v.detach() if k in ("gamma", "beta") else v.detach().bfloat16()).requires_grad_()
             for k, v in parameters(torch.float32).items()}
        x = torch.randn(2, 64, C, generator=torch.Generator().manual_seed(2)).cuda().bfloat16().requires_grad_()
        step(x, p, n, torch.ones_like(x), attention, norm)
        grads = [x.grad] + [v.grad for v in p.values()]
        assert all(torch.isfinite(t).all() for t in grads)
        first = first or grads
        assert all(torch.equal(a, b) for a, b in zip(first, grads))
