"""gsvdec_attention_forward / _backward against the formulas in 64 bits, with
bounds from the rounding units (attn_ref.py)."""
from __future__ import annotations

import pytest
import torch

from attn_ref import TYPES, check, reference

pytestmark = pytest.mark.gpu


def make(dtype, B, H, Hkv, Tq, Tk, D, w=-1, seed=0, heads_first=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[dtype]

    def rows(T, h):
        if heads_first:
            return torch.randn(B, h, T, D, generator=g, device="cuda").to(t)
        return torch.randn(B, T, h, D, generator=g, device="cuda").to(t).transpose(1, 2)

    x = {"q": rows(Tq, H), "k": rows(Tk, Hkv), "v": rows(Tk, Hkv), "do": rows(Tq, H)}
    if w >= 0:
        x["rel_k"] = (torch.randn(2 * w + 1, D, generator=g, device="cuda") * D ** -0.5).to(t)
        x["rel_v"] = (torch.randn(2 * w + 1, D, generator=g, device="cuda") * D ** -0.5).to(t)
    return x


def lengths(*n):
    return torch.tensor(n, dtype=torch.int32, device="cuda")


def run_and_check(gsv, x, **kw):
    rel = {n: x[n] for n in ("rel_k", "rel_v") if n in x}
    t = x["q"].dtype
    ref = reference(x["q"], x["k"], x["v"], x["do"], **kw, **rel)
    o, lse = gsv.attention(x["q"], x["k"], x["v"], **kw, **rel)
    check("o", o, ref, t)
    check("lse", lse, ref, torch.float32)
    grads = gsv.attention_backward(x["do"], x["q"], x["k"], x["v"], o, lse, **kw, **rel)
    for name, got in zip(("dq", "dk", "dv", "drel_k", "drel_v"), grads):
        if got is None:
            assert "rel_k" not in x
            continue
        assert got.dtype == t
        check(name, got, ref, t)
    gsv.ops_status()
    return o, lse, grads


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_head_widths(gsv, dtype, D):
    run_and_check(gsv, make(dtype, 2, 2, 2, 150, 150, D, w=4))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("D", [1, 7, 20, 72, 100, 127])
def test_odd_head_widths(gsv, dtype, D):
    run_and_check(gsv, make(dtype, 1, 2, 1, 70, 133, D, w=2), causal=True)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("T", [1, 2, 63, 64, 65, 127, 128, 129, 255, 257, 500])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths_around_tiles(gsv, dtype, T, causal):
    run_and_check(gsv, make(dtype, 1, 2, 2, T, T, 96, w=4), causal=causal)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("Tq,Tk", [(1, 300), (300, 1), (5, 700), (200, 61), (130, 257)])
@pytest.mark.parametrize("causal", [False, True])
def test_query_and_key_lengths_differ(gsv, dtype, Tq, Tk, causal):
    # With causal and Tq > Tk the first queries see no key.
    run_and_check(gsv, make(dtype, 2, 4, 2, Tq, Tk, 64, w=3), causal=causal)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("causal", [False, True])
def test_ragged_with_empty_sequences(gsv, dtype, causal):
    x = make(dtype, 6, 4, 2, 210, 190, 96, w=4)
    ql, kl = lengths(210, 0, 17, 130, 129, 1), lengths(190, 50, 0, 128, 129, 1)
    # What stands behind the last valid row must not matter.
    for n, name in ((ql, "q"), (ql, "do"), (kl, "k"), (kl, "v")):
        for b, m in enumerate(n.tolist()):
            x[name][b, :, m:] = float("nan")
    o, lse, (dq, dk, dv, _, _) = run_and_check(gsv, x, causal=causal, q_lengths=ql, k_lengths=kl)
    for b, m in enumerate(ql.tolist()):
        assert torch.all(o[b, :, m:] == 0) and torch.all(dq[b, :, m:] == 0)
        assert torch.all(lse[b, :, m:] == -float("inf"))
    for b, m in enumerate(kl.tolist()):
        assert torch.all(dk[b, :, m:] == 0) and torch.all(dv[b, :, m:] == 0)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("Tq,Tk,D", [(130, 1025, 96), (9, 2300, 64), (40, 1500, 128), (300, 900, 32)])
def test_long_keys_are_split_and_joined(gsv, dtype, Tq, Tk, D):
    # Few query tiles: the key tiles of one are dealt out to several blocks.
    x = make(dtype, 1, 2, 1, Tq, Tk, D, w=4)
    run_and_check(gsv, x, causal=True)
    run_and_check(gsv, x, q_lengths=lengths(Tq - 1), k_lengths=lengths(Tk // 2))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("H,Hkv,Tq", [(1, 1, 1), (8, 1, 1), (4, 2, 2), (3, 3, 7), (2, 1, 4)])
@pytest.mark.parametrize("D", [20, 32, 64, 128])
def test_few_queries(gsv, dtype, H, Hkv, Tq, D):
    x = make(dtype, 2, H, Hkv, Tq, 1000, D, w=2)
    run_and_check(gsv, x, causal=True, k_lengths=lengths(1000, 3))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("H,Hkv,Tq,D,w", [(8, 1, 1, 64, 15), (2, 1, 2, 96, 4), (1, 1, 8, 128, 15), (4, 2, 1, 33, 0)])
@pytest.mark.parametrize("causal", [False, True])
def test_few_queries_over_long_keys(gsv, dtype, H, Hkv, Tq, D, w, causal):
    # The keys are split over the largest clusters; the last ones, near the queries, over several of its blocks.
    run_and_check(gsv, make(dtype, 2, H, Hkv, Tq, 9001, D, w=w), causal=causal, k_lengths=lengths(9001, 8200))


def test_lengths_outside_the_tensor_are_clamped(gsv):
    x = make("bf16", 3, 2, 2, 50, 60, 32)
    run_and_check(gsv, x, q_lengths=lengths(-3, 50, 99), k_lengths=lengths(60, 1 << 30, -(1 << 31)))


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
@pytest.mark.parametrize("w", [0, 1, 7, 8, 15])
def test_windows(gsv, dtype, w):
    run_and_check(gsv, make(dtype, 2, 2, 1, 140, 140, 64, w=w), q_lengths=lengths(140, 9), k_lengths=lengths(140, 9))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("H,Hkv", [(8, 1), (6, 3), (5, 5)])
def test_shared_key_heads(gsv, dtype, H, Hkv):
    run_and_check(gsv, make(dtype, 2, H, Hkv, 90, 150, 64), causal=True)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_strides_and_alignment(gsv, dtype):
    # Heads first; a slice that starts off a 16-byte boundary; an odd row pitch; broadcast keys.
    run_and_check(gsv, make(dtype, 2, 3, 3, 75, 75, 64, w=2, heads_first=True))
    x = make(dtype, 2, 3, 3, 75, 80, 48)
    g = torch.Generator(device="cuda").manual_seed(5)
    wide = torch.randn(2, 75, 3, 49, generator=g, device="cuda").to(TYPES[dtype])
    x["q"] = wide[..., 1:].transpose(1, 2)
    x["k"] = x["k"][:1].expand(2, -1, -1, -1)
    x["v"] = x["v"][:, :1].expand(-1, 3, -1, -1)
    run_and_check(gsv, x)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_sharp_and_shifted_scores(gsv, dtype):
    # Rows whose maximum keeps rising along the keys, and scores far from 0.
    x = make(dtype, 1, 2, 2, 140, 400, 64)
    ramp = torch.linspace(0.2, 3.0, 400, device="cuda").view(1, 1, 400, 1)
    x["k"] = (x["k"].float() * ramp).to(TYPES[dtype])
    run_and_check(gsv, x, scale=0.5)
    x["q"] = (x["q"].float() + 2).to(TYPES[dtype])
    x["k"] = (x["k"].float() + 2).to(TYPES[dtype])
    run_and_check(gsv, x, scale=0.125)


@pytest.mark.parametrize("gain", [2.0 ** -10, 2.0 ** 9])
def test_fp16_gradients_of_any_size(gsv, gain):
    # ds spans many powers of two below do: none of it may be lost to fp16's range.
    x = make("fp16", 1, 2, 2, 300, 700, 64)
    x["do"] = (x["do"].float() * gain).to(torch.float16)
    if gain > 1:
        x["v"] = (x["v"].float() / 16).to(torch.float16)
    run_and_check(gsv, x)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_nothing_to_do(gsv, dtype):
    x = make(dtype, 2, 2, 2, 0, 40, 32, w=1)
    run_and_check(gsv, x)
    x = make(dtype, 2, 2, 2, 40, 0, 32, w=1)
    run_and_check(gsv, x)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("Tq,Tk,ql,kl", [(0, 40, 0, 40), (40, 0, 40, 0), (40, 40, 0, 40), (40, 40, 40, 0), (1, 1, 1, 0)])
def test_nothing_to_do_on_used_memory(gsv, dtype, Tq, Tk, ql, kl):
    # Workspace and outputs come from memory that held NaN.
    used = [torch.full((n,), float("nan"), device="cuda") for n in [64, 256, 1024, 4096, 16384, 65536, 1 << 20] * 6]
    x = make(dtype, 2, 2, 1, Tq, Tk, 40, w=1)
    del used
    run_and_check(gsv, x, q_lengths=lengths(ql, ql), k_lengths=lengths(kl, kl))


def test_infinite_scores_stay_in_their_row(gsv):
    x = make("bf16", 1, 1, 1, 140, 140, 64)
    x["q"][0, 0, 5] = float("inf")
    o, _ = gsv.attention(x["q"], x["k"], x["v"])
    bad = torch.isnan(o[0, 0]).any(-1).nonzero().flatten().tolist()
    assert bad == [5]


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_bits_repeat(gsv, dtype):
    x = make(dtype, 3, 4, 2, 333, 333, 96, w=4)
    kw = dict(rel_k=x["rel_k"], rel_v=x["rel_v"])
    first = None
    for _ in range(3):
        o, lse = gsv.attention(x["q"], x["k"], x["v"], **kw)
        out = (o, lse) + gsv.attention_backward(x["do"], x["q"], x["k"], x["v"], o, lse, **kw)
        first = first or out
        for a, b in zip(first, out):
            assert torch.equal(a, b)


def test_gradients_against_differences(gsv):
    # d/dh sum(o . do) of the fp32 forward against the gradients, in random directions.  The
    # quotient's error: O(h^2) of the third derivative plus the fp32 forward's rounding
    # (|do| |o| 2^-24 sqrt(n)) / h; with h = 2^-5 and unit inputs both stay below 2 % of the
    # gradient's size in a random direction.
    x = make("fp32", 1, 2, 1, 40, 50, 32, w=3)
    names = ("q", "k", "v", "rel_k", "rel_v")

    def value(y):
        return (gsv.attention(y["q"], y["k"], y["v"], rel_k=y["rel_k"], rel_v=y["rel_v"])[0].double()
                * x["do"].double()).sum()

    o, lse = gsv.attention(x["q"], x["k"], x["v"], rel_k=x["rel_k"], rel_v=x["rel_v"])
    grads = gsv.attention_backward(x["do"], x["q"], x["k"], x["v"], o, lse, rel_k=x["rel_k"], rel_v=x["rel_v"])
    for name, grad in zip(names, grads):
        d = torch.randn(x[name].shape, generator=torch.Generator().manual_seed(3)).cuda()
        d = d / d.norm()
        h = 2.0 ** -5
        up, down = dict(x), dict(x)
        up[name], down[name] = x[name] + h * d, x[name] - h * d
        quotient = (value(up) - value(down)) / (2 * h)
        slope = (grad.double() * d.double()).sum()
        assert abs(quotient - slope) <= 0.02 * grad.double().norm() / d.numel() ** 0.5 + 2e-4, name


def test_captured_and_on_another_stream(gsv):
    x = make("bf16", 2, 2, 2, 200, 200, 96, w=4)
    kw = dict(rel_k=x["rel_k"], rel_v=x["rel_v"], causal=True)

    def step():
        o, lse = gsv.attention(x["q"], x["k"], x["v"], **kw)
        return (o, lse) + gsv.attention_backward(x["do"], x["q"], x["k"], x["v"], o, lse, **kw)

    want = [t.clone() for t in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(want, side):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    new = make("bf16", 2, 2, 2, 200, 200, 96, w=4, seed=9)
    for n in ("q", "k", "v", "do", "rel_k", "rel_v"):
        x[n].copy_(new[n])
    graph.replay()
    got = [t.clone() for t in held]
    for a, b in zip(step(), got):
        assert torch.equal(a, b)


def test_refusals(gsv):
    x = make("bf16", 1, 2, 2, 8, 8, 32, w=1)
    q, k, v = x["q"], x["k"], x["v"]
    for bad in (dict(k=k.float()), dict(k=k[:, :, :, :16]), dict(v=v.cpu()), dict(q=q.transpose(-1, -2)),
                dict(q=q.double(), k=k.double(), v=v.double())):
        y = {"q": q, "k": k, "v": v, **bad}
        with pytest.raises(ValueError):
            gsv.attention(y["q"], y["k"], y["v"])
    with pytest.raises(ValueError):
        gsv.attention(q, k, v, rel_k=x["rel_k"])
    with pytest.raises(ValueError):
        gsv.attention(q, k, v, k_lengths=torch.ones(1, dtype=torch.int64, device="cuda"))
    for kw in (dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf"))):
        with pytest.raises(gsv.GsvDecError) as e:
            gsv.attention(q, k, v, **kw)
        assert e.value.status == "GSV_E_INVALID_ARG"
    big = torch.zeros(1, 1, 4, 136, device="cuda")
    with pytest.raises(gsv.GsvDecError):
        gsv.attention(big, big, big)
    with pytest.raises(gsv.GsvDecError):
        gsv.attention(q[:, :1].expand(-1, 3, -1, -1), k, v)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("Tq,Tk,ql,kl", [(200, 61, (200, 150), (61, 10)), (333, 300, (333, 300), (70, 300)),
                                         (6, 3, (6, 5), (3, 0))])
@pytest.mark.parametrize("w", [-1, 3])
def test_queries_without_a_key_hold_anything(gsv, dtype, Tq, Tk, ql, kl, w):
    # With causal the first ql - kl queries see no key: they add nothing to any gradient, whatever they hold.
    x = make(dtype, 2, 4, 2, Tq, Tk, 64, w=w)
    for b in range(2):
        n = ql[b] - kl[b]
        x["q"][b, :, :n] = x["do"][b, :, :n] = 0
    kw = dict(causal=True, q_lengths=lengths(*ql), k_lengths=lengths(*kl))
    want = run_and_check(gsv, x, **kw)
    for bad in (float("nan"), float("inf")):
        for b in range(2):
            n = ql[b] - kl[b]
            x["q"][b, :, :n] = bad
            x["do"][b, :, :n] = -bad
        kw2 = dict(kw, **{n: x[n] for n in ("rel_k", "rel_v") if n in x})
        o, lse = gsv.attention(x["q"], x["k"], x["v"], **kw2)
        grads = gsv.attention_backward(x["do"], x["q"], x["k"], x["v"], o, lse, **kw2)
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
        for a, b in zip(grads, want[2]):
            assert (a is None and b is None) or torch.equal(a, b)


def test_heads_without_channels_are_refused(gsv):
    q = torch.zeros(1, 2, 4, 0, device="cuda")
    for kw in ({}, dict(scale=1.0)):
        with pytest.raises(gsv.GsvDecError) as e:
            gsv.attention(q, q, q, **kw)
        assert e.value.status == "GSV_E_INVALID_ARG"


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("Tq,Tk", [(70, 90), (1, 1), (200, 0)])
@pytest.mark.parametrize("causal", [False, True])
def test_queries_of_an_utterance_without_keys_hold_anything(gsv, dtype, Tq, Tk, causal):
    x = make(dtype, 3, 4, 2, Tq, Tk, 48, w=4)
    x["q"][1] = x["do"][1] = 0
    kw = dict(causal=causal, k_lengths=lengths(Tk, 0, Tk), rel_k=x["rel_k"], rel_v=x["rel_v"])
    want = run_and_check(gsv, x, **{n: v for n, v in kw.items() if not n.startswith("rel")})
    x["q"][1], x["do"][1] = float("nan"), float("inf")
    if Tk == 0:
        x["q"][:], x["do"][:] = float("nan"), float("nan")
    o, lse = gsv.attention(x["q"], x["k"], x["v"], **kw)
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    for a, b in zip(gsv.attention_backward(x["do"], x["q"], x["k"], x["v"], o, lse, **kw), want[2]):
        assert torch.equal(a, b)
