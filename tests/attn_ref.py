"""Attention with relative keys and values in 64 bits, with its gradients and
bounds on the rounding errors of an implementation.

The bounds follow an evaluation with fp32 sums (unit U = 2^-24; a factor 2
covers sums that truncate instead of rounding) and, for 16-bit inputs,
probabilities, ds and o rounded to the inputs' type once (unit ut = eps / 2).
To first order, with |x| the absolute values:

  s:      es = 2 (D + 8) U scale |q||k|, plus 2 U |s| for its scaling and the
          exponent's argument against the row's maximum or log-sum-exp
  p:      relative ep = 2 max_j es + (n + 16) 2 U (numerator and sum)
  o:      sum p |v| (ep + ut + 2 (n + 8) U) + ut |o|
  ds:     p |dp - delta| (ep + ut) + p (2 D U |do||v| + (ut + 2 D U) |do||o|)
  dq:     scale sum |eds| |k| + scale 2 (n + 8) U sum |ds| |k| + ut |dq|
  dk, dv, drel likewise over the rows they sum.
"""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def unit(t):
    return torch.finfo(t).eps / 2


def geometry(B, Tq, Tk, q_lengths, k_lengths, causal, dev):
    ql = torch.full((B,), Tq) if q_lengths is None else torch.as_tensor(q_lengths).cpu().clamp(0, Tq)
    kl = torch.full((B,), Tk) if k_lengths is None else torch.as_tensor(k_lengths).cpu().clamp(0, Tk)
    ql, kl = ql.long().to(dev).view(B, 1, 1, 1), kl.long().to(dev).view(B, 1, 1, 1)
    i = torch.arange(Tq, device=dev).view(1, 1, Tq, 1)
    j = torch.arange(Tk, device=dev).view(1, 1, 1, Tk)
    r = j - (i + kl - ql)
    ok = (i < ql) & (j < kl)
    return (ok & (r <= 0) if causal else ok), r


def reference(q, k, v, do=None, scale=None, causal=False, q_lengths=None, k_lengths=None, rel_k=None, rel_v=None):
    """dict of results ("o", "lse", "dq", ...) in fp64, and of bounds ("e_o", ...)."""
    t, dev = q.dtype, q.device
    B, H, Tq, D = q.shape
    Hkv, Tk = k.shape[1:3]
    g = H // Hkv
    scale = 1 / math.sqrt(D) if scale is None else scale
    ut = 0.0 if t == torch.float32 else unit(t)
    uo = unit(t)
    ok, r = geometry(B, Tq, Tk, q_lengths, k_lengths, causal, dev)
    w = -1 if rel_k is None else rel_k.shape[0] // 2
    near = (r.abs() <= w) & ok
    idx = (r + w).clamp(0, max(2 * w, 0))

    def clean(x, n, T):  # rows past the length hold anything
        x = x.double()
        if n is None:
            return x
        n = torch.as_tensor(n).to(dev).long().clamp(0, T)
        return torch.where(torch.arange(T, device=dev).view(1, 1, T, 1) < n.view(B, 1, 1, 1), x, 0.0)

    q = clean(q, q_lengths, Tq)
    k, v = (clean(x, k_lengths, Tk).repeat_interleave(g, 1) for x in (k, v))
    rk, rv = (None, None) if w < 0 else (rel_k.double(), rel_v.double())

    def gather(rows, rel):  # rows . rel by offset
        return torch.where(near, (rows @ rel.T).gather(-1, idx.expand(B, H, Tq, Tk)), 0.0)

    def band(x):
        return torch.stack([torch.where(near & (r == o), x, 0.0).sum(-1) for o in range(-w, w + 1)], -1)

    s = q @ k.transpose(-1, -2)
    sa = q.abs() @ k.abs().transpose(-1, -2)
    if w >= 0:
        s, sa = s + gather(q, rk), sa + gather(q.abs(), rk.abs())
    s = (s * scale).masked_fill(~ok, -math.inf)
    m = s.amax(-1, keepdim=True) if Tk else torch.full((B, H, Tq, 1), -math.inf, dtype=torch.float64, device=dev)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(s - m)
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l == 0, 1.0, l)
    lse = (m + torch.log(l)).squeeze(-1)
    n = ok.sum(-1, keepdim=True).double()
    big = torch.where(ok, s.abs(), 0.0)
    es = torch.where(ok, 2 * (D + 8) * U * scale * sa + 4 * U * big, 0.0)
    es_row = es.amax(-1, keepdim=True) + 4 * U * big.amax(-1, keepdim=True) if Tk else n
    ep = 2 * es_row + 2 * (n + 16) * U
    out = {"o": p @ v, "lse": lse}
    pv = p @ v.abs()
    if w >= 0:
        bp = band(p)
        out["o"] = out["o"] + bp @ rv
        pv = pv + bp @ rv.abs()
    out["e_o"] = pv * (ep + ut + 2 * (n + 8) * U) + uo * out["o"].abs()
    out["e_lse"] = (es_row + 2 * (n + 16) * U).squeeze(-1) + U * torch.where(lse == -math.inf, 0.0, lse.abs())
    if do is None:
        return out
    do = clean(do, q_lengths, Tq)
    o = out["o"]
    dp, dpa = do @ v.transpose(-1, -2), do.abs() @ v.abs().transpose(-1, -2)
    if w >= 0:
        dp, dpa = dp + gather(do, rv), dpa + gather(do.abs(), rv.abs())
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    eds = p * ((dp - delta).abs() * (ep + ut) + 2 * (D + 8) * U * dpa
               + (ut + 2 * (D + 8) * U) * (do.abs() * o.abs()).sum(-1, keepdim=True))
    acc = 2 * (n + 8) * U
    fold = lambda x: x.view(B, Hkv, g, Tk, D).sum(2)  # noqa: E731
    rows = 2 * (g * Tq + 8) * U
    dsT, edsT, pT = ds.transpose(-1, -2), eds.transpose(-1, -2), p.transpose(-1, -2)
    dq, edq = ds @ k, eds @ k.abs() + acc * (ds.abs() @ k.abs())
    if w >= 0:
        bs, ebs = band(ds), band(eds)
        dq = dq + bs @ rk
        edq = edq + ebs @ rk.abs() + acc * (bs.abs() @ rk.abs())
        N = 2 * (B * H * Tq + 8) * U
        e = "bhtr,bhtd->rd"
        out["drel_k"] = scale * torch.einsum(e, bs, q)
        out["e_drel_k"] = scale * (torch.einsum(e, ebs, q.abs()) + N * torch.einsum(e, bs.abs(), q.abs())) \
            + uo * out["drel_k"].abs()
        out["drel_v"] = torch.einsum(e, bp, do)
        out["e_drel_v"] = torch.einsum(e, bp * (ep + ut + N), do.abs()) + uo * out["drel_v"].abs()
    out["dq"] = scale * dq
    out["e_dq"] = scale * edq + uo * out["dq"].abs()
    out["dk"] = scale * fold(dsT @ q)
    out["e_dk"] = scale * fold(edsT @ q.abs() + rows * (dsT.abs() @ q.abs())) + uo * out["dk"].abs()
    out["dv"] = fold(pT @ do)
    out["e_dv"] = fold((p * (ep + ut + rows)).transpose(-1, -2) @ do.abs()) + uo * out["dv"].abs()
    return out


def check(name, got, ref, t):
    """|got - ref| within the bound; half a step of the type's subnormals is added."""
    want, bound = ref[name], ref["e_" + name]
    got = got.double()
    assert got.shape == want.shape, name
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fin), f"{name}: finite values in other places"
    assert torch.equal(got[~fin], want[~fin]), f"{name}: other infinities"
    tiny = 2.0 ** -24 if t == torch.float16 else 0.0  # fp16 steps 2^-24 below 2^-14, twice on a result's way
    over = ((got - want).abs() - bound - tiny)[fin]
    assert over.numel() == 0 or over.max() <= 0, \
        f"{name}: off by {(got - want).abs()[fin].max():.3e}, {over.max():.3e} over the bound"
