"""Cases of the text encoder's attention and residual norm, with their gradients.

Four operators are covered, each as a plain torch form and as the library's call:

``attn_fwd``   o = softmax(scale q k^T + relative terms) v, with its log-sum-exp
``attn_bwd``   the gradients of q, k, v and of the relative keys and values
``norm_fwd``   LayerNorm over channels of x + y, with its mean and 1 / deviation
``norm_bwd``   the gradients of x (+ y), gamma and beta

Attention tensors are [B, H, T, D] views of time-major [B, T, H, D] storage, as
the library's projections leave them.  ``lengths`` give the valid frames of
each utterance; the sequences are aligned at their ends, so query i of
utterance b stands at key position i + k_len[b] - q_len[b].  ``window`` = w adds
the encoder's learned relative keys and values for the offsets -w .. w
(-1: none).
"""
import math
import random

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# -- the cases ------------------------------------------------------------------

def _attn(name, op, dtype, B, H, Hkv, Tq, Tk, D, window=-1, causal=False, ragged=False, empty=False):
    return {"name": name, "op": op, "dtype": dtype, "B": B, "H": H, "Hkv": Hkv, "Tq": Tq, "Tk": Tk, "D": D,
            "window": window, "causal": causal, "ragged": ragged, "empty": empty}


def _norm(name, op, dtype, layout, B, C, T, residual=True, ragged=False):
    return {"name": name, "op": op, "dtype": dtype, "layout": layout, "B": B, "C": C, "T": T,
            "residual": residual, "ragged": ragged}


def listed():
    return [
        # One short sentence through the text encoder (192 channels, 2 heads of 96, window 4).
        _attn("attn_fwd_sentence_fp32", "attn_fwd", "fp32", 1, 2, 2, 37, 37, 96, window=4),
        # A training or batch-serving step of the encoder on 16 utterances of up to 10 s.
        _attn("attn_fwd_encoder_bf16", "attn_fwd", "bf16", 16, 2, 2, 500, 500, 96, window=4, ragged=True),
        # A long causal sequence, 16 heads of 64.
        _attn("attn_fwd_long_causal_bf16", "attn_fwd", "bf16", 4, 16, 16, 4096, 4096, 64, causal=True),
        # One token a sequence against its cached keys, 16 heads of 32 over 4 shared key heads.
        _attn("attn_fwd_token_fp16", "attn_fwd", "fp16", 16, 16, 4, 1, 1531, 32, causal=True, ragged=True),
        # The encoder's training step, backward, relative keys and values included.
        _attn("attn_bwd_encoder_bf16", "attn_bwd", "bf16", 16, 2, 2, 500, 500, 96, window=4, ragged=True),
        # Cross-attention of audio frames to phonemes in full precision, 4 heads of 128.
        _attn("attn_bwd_cross_fp32", "attn_bwd", "fp32", 4, 4, 4, 500, 173, 128, ragged=True),
        # The long causal sequence, backward.
        _attn("attn_bwd_long_causal_bf16", "attn_bwd", "bf16", 2, 16, 16, 4096, 4096, 64, causal=True),
        # The norm after one short sentence's attention, in the encoder's [B, C, T] layout.
        _norm("norm_fwd_sentence_fp32", "norm_fwd", "fp32", "bct", 1, 192, 37),
        # The norm of wide rows, time-major.
        _norm("norm_fwd_rows_bf16", "norm_fwd", "bf16", "btc", 8, 1024, 4096),
        # The encoder's training step, 64 utterances of up to 10 s.
        _norm("norm_bwd_encoder_fp32", "norm_bwd", "fp32", "bct", 64, 192, 500, ragged=True),
        # Odd rows: no row but the first starts on a vector's boundary.
        _norm("norm_bwd_odd_fp16", "norm_bwd", "fp16", "btc", 3, 515, 1001, residual=False, ragged=True),
        # Wide rows, backward.
        _norm("norm_bwd_rows_bf16", "norm_bwd", "bf16", "btc", 8, 1024, 4096),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["attn_fwd", "attn_fwd", "attn_bwd", "attn_bwd", "norm_fwd", "norm_bwd"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op.startswith("norm"):
        B, C = _log(rng, 1, 64), _log(rng, 64, 2048)
        T = _log(rng, 1, max(2, min(4096, (1 << 25) // (B * C))))
        c = _norm("", op, dtype, rng.choice(["bct", "btc"]), B, C, T, rng.random() < 0.7, rng.random() < 0.5)
        del c["name"]
        return c
    D = rng.choice([32, 64, 64, 96, 96, 128])
    Hkv = _log(rng, 1, 8)
    H = Hkv * rng.choice([1, 1, 2, 4])
    B = _log(rng, 1, 16)
    kind = rng.choice(["self", "self", "cross", "token"]) if op == "attn_fwd" else rng.choice(["self", "self", "cross"])
    top = _attn("", "attn_bwd", "bf16", 2, 16, 16, 4096, 4096, 64, causal=True)
    room = work(top)["flops"] / (10.0 * D * B * H) / (8 if dtype == "fp32" else 1)
    if kind == "token":
        Tq, Tk = 1, _log(rng, 1, min(16384, int((1 << 28) // (B * Hkv * D))))
    else:
        Tk = _log(rng, 2, max(3, min(4096, int(math.sqrt(room)))))
        Tq = Tk if kind == "self" else _log(rng, 2, max(3, min(4096, int(math.sqrt(room)))))
    c = _attn("", op, dtype, B, H, Hkv, Tq, Tk, D, window=4 if kind == "self" and rng.random() < 0.6 else -1,
              causal=kind != "cross" and rng.random() < 0.5, ragged=rng.random() < 0.6, empty=rng.random() < 0.2)
    del c["name"]
    return c


# -- inputs ---------------------------------------------------------------------

def _spread(n, T, ragged, empty=False):
    """Lengths between two fifths of T and T, evenly spread; the last one 0 where empty."""
    if not ragged:
        return [T] * n
    lens = [max(1, T - (T * 3 * b) // (5 * n)) for b in range(n)]
    if empty and n > 1:
        lens[-1] = 0
    return lens


def _lens(case, which):
    if case["op"].startswith("norm"):
        return _spread(case["B"], case["T"], case["ragged"])
    if which == "q" and case["Tq"] == 1:
        return [1] * case["B"]
    T = case["Tq"] if which == "q" else case["Tk"]
    return _spread(case["B"], T, case["ragged"], case["empty"])


def _ramp(case):
    """The utterances' order: q and k lengths of one utterance stay together."""
    return list(zip(_lens(case, "q"), _lens(case, "k")))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 2 + 1)
    dev, dt = "cuda", TYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(shape, generator=gen, device=dev) * std).to(dtype)

    order = list(range(case["B"]))
    random.Random(seed).shuffle(order)
    st = {"case": case}
    if case["op"].startswith("norm"):
        B, C, T = case["B"], case["C"], case["T"]
        shape = (B, C, T) if case["layout"] == "bct" else (B, T, C)
        lens = _lens(case, "q")
        st["lengths"] = torch.tensor([lens[i] for i in order], dtype=torch.int32, device=dev) if case["ragged"] else None
        st["x"] = normal(*shape) + 0.25
        st["y"] = normal(*shape, std=0.5) if case["residual"] else None
        st["gamma"] = 1.0 + normal(C, std=0.1, dtype=torch.float32)
        st["beta"] = normal(C, std=0.1, dtype=torch.float32)
        if case["op"] == "norm_bwd":
            st["dout"] = normal(*shape)
            _, st["mean"], st["rstd"] = _plain_norm_fwd(st)
        return st
    B, H, Hkv, Tq, Tk, D = (case[k] for k in ("B", "H", "Hkv", "Tq", "Tk", "D"))
    pairs = _ramp(case)
    ql, kl = [pairs[i][0] for i in order], [pairs[i][1] for i in order]
    st["q_lengths"] = torch.tensor(ql, dtype=torch.int32, device=dev) if case["ragged"] and Tq > 1 else None
    st["k_lengths"] = torch.tensor(kl, dtype=torch.int32, device=dev) if case["ragged"] else None
    st["q"] = normal(B, Tq, H, D).transpose(1, 2)
    st["k"] = normal(B, Tk, Hkv, D).transpose(1, 2)
    st["v"] = normal(B, Tk, Hkv, D).transpose(1, 2)
    w = case["window"]
    st["rel_k"] = normal(2 * w + 1, D, std=D ** -0.5) if w >= 0 else None
    st["rel_v"] = normal(2 * w + 1, D, std=D ** -0.5) if w >= 0 else None
    if case["op"] == "attn_bwd":
        st["do"] = normal(B, Tq, H, D).transpose(1, 2)
        o, st["lse"] = _plain_attn_fwd(st)
        st["o"] = o.transpose(1, 2).contiguous().transpose(1, 2)
    return st


# -- the plain forms ------------------------------------------------------------

def _attn_tables(st):
    """(allowed [B, 1, Tq, Tk], distance key - query position [B, 1, Tq, Tk])."""
    case, q, k = st["case"], st["q"], st["k"]
    B, Tq, Tk = case["B"], case["Tq"], case["Tk"]
    i = torch.arange(Tq, device=q.device).view(1, 1, Tq, 1)
    j = torch.arange(Tk, device=q.device).view(1, 1, 1, Tk)
    full = lambda n, t: torch.full((B,), n, device=q.device) if t is None else t.long()  # noqa: E731
    ql = full(Tq, st["q_lengths"]).view(B, 1, 1, 1)
    kl = full(Tk, st["k_lengths"]).view(B, 1, 1, 1)
    dist = j - (i + kl - ql)
    ok = (i < ql) & (j < kl)
    if case["causal"]:
        ok = ok & (dist <= 0)
    return ok, dist


def _attn_probs(st):
    case = st["case"]
    g = case["H"] // case["Hkv"]
    q = st["q"].float()
    k = st["k"].float().repeat_interleave(g, 1)
    ok, dist = _attn_tables(st)
    s = q @ k.transpose(-1, -2)
    w = case["window"]
    if w >= 0:
        rel = q @ st["rel_k"].float().t()
        near = dist.abs() <= w
        s = s + torch.where(near, rel.gather(-1, (dist + w).clamp(0, 2 * w).expand(s.shape)), 0.0)
    s = (s * case["D"] ** -0.5).masked_fill(~ok, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(s - m)
    l = p.sum(-1, keepdim=True)
    return p / torch.where(l == 0, 1.0, l), (m + torch.log(l)).squeeze(-1), dist


def _band(p, dist, w):
    """p summed by its offset: [B, H, Tq, 2 w + 1]."""
    return torch.stack([torch.where(dist == r, p, 0.0).sum(-1) for r in range(-w, w + 1)], -1)


def _plain_attn_fwd(st):
    case = st["case"]
    p, lse, dist = _attn_probs(st)
    o = p @ st["v"].float().repeat_interleave(case["H"] // case["Hkv"], 1)
    if case["window"] >= 0:
        o = o + _band(p, dist, case["window"]) @ st["rel_v"].float()
    return o.to(st["q"].dtype), lse


def _plain_attn_bwd(st):
    case = st["case"]
    B, H, Hkv, Tq, Tk, D = (case[k] for k in ("B", "H", "Hkv", "Tq", "Tk", "D"))
    g, w, scale, dt = H // Hkv, case["window"], D ** -0.5, st["q"].dtype
    q, do = st["q"].float(), st["do"].float()
    k, v = (st[n].float().repeat_interleave(g, 1) for n in ("k", "v"))
    p, _, dist = _attn_probs(st)
    dp = do @ v.transpose(-1, -2)
    if w >= 0:
        rel = do @ st["rel_v"].float().t()
        dp = dp + torch.where(dist.abs() <= w, rel.gather(-1, (dist + w).clamp(0, 2 * w).expand(dp.shape)), 0.0)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta) * scale
    dq = ds @ k
    dk = (ds.transpose(-1, -2) @ q).view(B, Hkv, g, Tk, D).sum(2)
    dv = (p.transpose(-1, -2) @ do).view(B, Hkv, g, Tk, D).sum(2)
    if w < 0:
        return dq.to(dt), dk.to(dt), dv.to(dt)
    bp, bs = _band(p, dist, w), _band(ds, dist, w)
    dq = dq + bs @ st["rel_k"].float()
    drk = torch.einsum("bhtr,bhtd->rd", bs, q)
    drv = torch.einsum("bhtr,bhtd->rd", bp, do)
    return dq.to(dt), dk.to(dt), dv.to(dt), drk.to(dt), drv.to(dt)


def _norm_parts(st):
    """(x + y as [B, T, C] in 32 bits, valid frames [B, T, 1])."""
    x = st["x"].float()
    if st["y"] is not None:
        x = x + st["y"].float()
    if st["case"]["layout"] == "bct":
        x = x.transpose(1, 2)
    B, T, _ = x.shape
    t = torch.arange(T, device=x.device).view(1, T, 1)
    n = st["lengths"]
    ok = t < (T if n is None else n.view(B, 1, 1))
    return x, ok.expand(B, T, 1)


def _like(st, t):
    t = t.transpose(1, 2) if st["case"]["layout"] == "bct" else t
    return t.to(st["x"].dtype).contiguous()


def _plain_norm_fwd(st):
    x, ok = _norm_parts(st)
    mean = x.mean(-1, keepdim=True)
    rstd = torch.rsqrt(((x - mean) ** 2).mean(-1, keepdim=True) + 1e-5)
    out = torch.where(ok, (x - mean) * rstd * st["gamma"] + st["beta"], 0.0)
    zero = lambda t: torch.where(ok, t, 0.0).squeeze(-1)  # noqa: E731
    return _like(st, out), zero(mean), zero(rstd)


def _plain_norm_bwd(st):
    x, ok = _norm_parts(st)
    dout = st["dout"].float()
    if st["case"]["layout"] == "bct":
        dout = dout.transpose(1, 2)
    dout = torch.where(ok, dout, 0.0)
    mean, rstd = st["mean"].unsqueeze(-1), st["rstd"].unsqueeze(-1)
    xh = torch.where(ok, (x - mean) * rstd, 0.0)
    a = dout * st["gamma"]
    dx = rstd * (a - a.mean(-1, keepdim=True) - xh * (a * xh).mean(-1, keepdim=True))
    dgamma = (dout * xh).sum((0, 1), dtype=torch.float64).float()
    dbeta = dout.sum((0, 1), dtype=torch.float64).float()
    return _like(st, dx), dgamma, dbeta


# -- one pass -------------------------------------------------------------------

def run(st):
    op = st["case"]["op"]
    if not own:
        return {"attn_fwd": _plain_attn_fwd, "attn_bwd": _plain_attn_bwd, "norm_fwd": _plain_norm_fwd,
                "norm_bwd": _plain_norm_bwd}[op](st)
    from __graft_entry__ import load_package

    gsv = load_package()
    case = st["case"]
    if op == "norm_fwd":
        return gsv.add_norm(st["x"], st["y"], st["gamma"], st["beta"], lengths=st["lengths"], layout=case["layout"])
    if op == "norm_bwd":
        return gsv.add_norm_backward(st["dout"], st["x"], st["y"], st["gamma"], st["mean"], st["rstd"],
                                     lengths=st["lengths"], layout=case["layout"])
    opts = dict(causal=case["causal"], q_lengths=st["q_lengths"], k_lengths=st["k_lengths"], rel_k=st["rel_k"],
                rel_v=st["rel_v"])
    if op == "attn_fwd":
        return gsv.attention(st["q"], st["k"], st["v"], **opts)
    grads = gsv.attention_backward(st["do"], st["q"], st["k"], st["v"], st["o"], st["lse"], **opts)
    return grads if case["window"] >= 0 else grads[:3]


# -- what a pass cannot do without ----------------------------------------------

def _pairs(case):
    n = 0
    for ql, kl in _ramp(case):
        if case["causal"]:
            first = max(0, ql - kl)  # queries before it see no key
            rows = ql - first
            n += rows * (kl - ql + first + 1 + kl) // 2
        else:
            n += ql * kl
    return n


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"].startswith("norm"):
        frames = sum(_lens(case, "q"))
        n, total = frames * case["C"], case["B"] * case["T"] * case["C"]
        reads = (2 if case["residual"] else 1) + (case["op"] == "norm_bwd")
        return {"bytes": reads * n * e + total * e + 8 * frames + 8 * case["C"],
                "flops": (8 if case["op"] == "norm_fwd" else 14) * n}
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    tq = sum(q for q, _ in _ramp(case))
    tk = sum(k for _, k in _ramp(case))
    allq, allk = case["B"] * case["Tq"], case["B"] * case["Tk"]
    rel = 2 * (2 * case["window"] + 1) * D if case["window"] >= 0 else 0
    if case["op"] == "attn_fwd":
        return {"bytes": e * D * (tq * H + 2 * tk * Hkv + allq * H) + e * rel + 4 * H * allq,
                "flops": 4 * D * H * _pairs(case)}
    return {"bytes": e * D * (3 * tq * H + 2 * tk * Hkv + allq * H + 2 * allk * Hkv) + 2 * e * rel + 4 * H * tq,
            "flops": 10 * D * H * _pairs(case)}


# -- the definition in 64 bits --------------------------------------------------

def _exact_norm(case, st):
    d = torch.float64
    cl = case["layout"] == "btc"
    x = st["x"].to(d) + (0 if st["y"] is None else st["y"].to(d))
    x = x if cl else x.permute(0, 2, 1)
    B, T, C = x.shape
    lens = [T] * B if st["lengths"] is None else st["lengths"].tolist()
    mean = x.sum(2) / C
    rstd = 1.0 / torch.sqrt(((x - mean[:, :, None]) ** 2).sum(2) / C + 1e-5)
    for b, n in enumerate(lens):
        mean[b, n:] = 0
        rstd[b, n:] = 0
    gamma = st["gamma"].to(d)
    xh = (x - mean[:, :, None]) * rstd[:, :, None]
    back = (lambda t: t) if cl else (lambda t: t.permute(0, 2, 1).contiguous())
    if case["op"] == "norm_fwd":
        out = xh * gamma + st["beta"].to(d)
        for b, n in enumerate(lens):
            out[b, n:] = 0
        return back(out), mean, rstd
    g = st["dout"].to(d)
    g = (g if cl else g.permute(0, 2, 1)).clone()
    for b, n in enumerate(lens):
        g[b, n:] = 0
    gg = g * gamma
    dx = (gg - gg.sum(2, keepdim=True) / C - xh * ((gg * xh).sum(2, keepdim=True) / C)) * rstd[:, :, None]
    return back(dx), (g * xh).flatten(0, 1).sum(0), g.flatten(0, 1).sum(0)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"].startswith("norm"):
        return _exact_norm(case, st)
    d, dev = torch.float64, st["q"].device
    B, H, Hkv, Tq, Tk, D, w = (case[k] for k in ("B", "H", "Hkv", "Tq", "Tk", "D", "window"))
    bwd, group, scale = case["op"] == "attn_bwd", H // Hkv, 1.0 / math.sqrt(D)
    ql = [Tq] * B if st["q_lengths"] is None else st["q_lengths"].tolist()
    kl = [Tk] * B if st["k_lengths"] is None else st["k_lengths"].tolist()
    o = torch.zeros(B, H, Tq, D, dtype=d, device=dev)
    lse = torch.full((B, H, Tq), -math.inf, dtype=d, device=dev)
    dq, dk, dv = torch.zeros_like(o), *(torch.zeros(B, Hkv, Tk, D, dtype=d, device=dev) for _ in range(2))
    rk, rv = (st[n].to(d) if w >= 0 else None for n in ("rel_k", "rel_v"))
    drk, drv = (torch.zeros(2 * max(w, 0) + 1, D, dtype=d, device=dev) for _ in range(2))
    for b in range(B):
        n, m = ql[b], kl[b]
        if n == 0 or m == 0:
            continue
        pos = torch.arange(n, device=dev)[:, None] + (m - n)
        off = torch.arange(m, device=dev)[None, :] - pos
        rows = (off <= 0).any(1) if case["causal"] else torch.ones(n, dtype=torch.bool, device=dev)
        for h in range(H):
            q, k, v = st["q"][b, h, :n].to(d), st["k"][b, h // group, :m].to(d), st["v"][b, h // group, :m].to(d)
            s = q @ k.T
            for r in range(-w, w + 1):
                s = s + (off == r) * (q @ rk[r + w])[:, None]
            s = s * scale
            if case["causal"]:
                s = s.masked_fill(off > 0, -math.inf)
            z = torch.logsumexp(s, 1)
            p = torch.exp(s - torch.where(rows, z, 0.0)[:, None])
            lse[b, h, :n] = z
            if not bwd:
                o[b, h, :n] = p @ v
                for r in range(-w, w + 1):
                    o[b, h, :n] += ((off == r) * p).sum(1)[:, None] * rv[r + w]
                continue
            g = st["do"][b, h, :n].to(d)
            gp = g @ v.T
            for r in range(-w, w + 1):
                gp = gp + (off == r) * (g @ rv[r + w])[:, None]
            gs = p * (gp - (p * gp).sum(1, keepdim=True)) * scale
            dv[b, h // group, :m] += p.T @ g
            dk[b, h // group, :m] += gs.T @ q
            dq[b, h, :n] = gs @ k
            for r in range(-w, w + 1):
                near = off == r
                dq[b, h, :n] += (near * gs).sum(1)[:, None] * rk[r + w]
                drk[r + w] += (near * gs).sum(1) @ q
                drv[r + w] += (near * p).sum(1) @ g
    if not bwd:
        return o, lse
    return (dq, dk, dv, drk, drv) if w >= 0 else (dq, dk, dv)
