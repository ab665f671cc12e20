"""gsvdec_norm_forward / _backward against the formulas in 64 bits.

Bounds, U = 2^-24, ut the half step of the outputs' type: a frame's mean is a
sum of C values (error 2 (C + 8) U mean|s|), the deviation's square another;
xh = (s - mean) rstd is then off by eh = rstd (2 (C + 8) U mean|s| + 4 U |s|) +
|xh| 2 (C + 8) U, and the results follow by the product rule.
"""
from __future__ import annotations

import pytest
import torch

from attn_ref import TYPES, U, unit

pytestmark = pytest.mark.gpu


def make(dtype, layout, B, C, T, y=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (B, C, T) if layout == "bct" else (B, T, C)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    t = TYPES[dtype]
    return {"x": (r(*shape) + 0.5).to(t), "y": r(*shape).to(t) if y else None, "gamma": 1 + 0.2 * r(C),
            "beta": 0.2 * r(C), "d_out": r(*shape).to(t)}


def reference(x, layout, lengths, eps=1e-5):
    rows = (lambda t: t.double().transpose(1, 2)) if layout == "bct" else (lambda t: t.double())
    s = rows(x["x"]) + (0 if x["y"] is None else rows(x["y"]))
    B, T, C = s.shape
    t = x["x"].dtype
    ut = unit(t)
    ok = torch.ones(B, T, 1, dtype=torch.bool, device=s.device)
    if lengths is not None:
        ok = torch.arange(T, device=s.device).view(1, T, 1) < lengths.view(B, 1, 1)
    s = torch.where(ok, s, 0.0)
    mean = s.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((s - mean) ** 2).mean(-1, keepdim=True) + eps)
    g = 2 * (C + 8) * U
    em = g * s.abs().mean(-1, keepdim=True) + U * mean.abs()
    er = rstd * (g + 2 * rstd * em)
    xh = (s - mean) * rstd
    eh = rstd * (em + 4 * U * s.abs()) + xh.abs() * (er / rstd + 4 * U)
    gamma, beta = x["gamma"].double(), x["beta"].double()
    z = lambda v: torch.where(ok, v, 0.0)  # noqa: E731
    back = (lambda v: v.transpose(1, 2)) if layout == "bct" else (lambda v: v)
    out = z(xh * gamma + beta)
    e_out = z(eh * gamma.abs() + 4 * U * (xh * gamma).abs() + 4 * U * out.abs() + ut * out.abs())
    d = z(rows(x["d_out"]))
    a = d * gamma
    m0, m1 = a.mean(-1, keepdim=True), (a * xh).mean(-1, keepdim=True)
    dx = z(rstd * (a - m0 - xh * m1))
    size = a.abs() + a.abs().mean(-1, keepdim=True) + xh.abs() * (a * xh).abs().mean(-1, keepdim=True)
    e_dx = rstd * ((g + 8 * U) * size + eh * (a * xh).abs().mean(-1, keepdim=True)
                   + xh.abs() * (a.abs() * eh).mean(-1, keepdim=True)) + er * size + ut * dx.abs()
    n = 2 * (B * T + 8) * U
    res = {"out": (back(out), back(e_out)), "mean": (z(mean)[..., 0], z(em)[..., 0]),
           "rstd": (z(rstd)[..., 0], z(er + 4 * U * rstd)[..., 0]), "dx": (back(dx), back(z(e_dx))),
           "dgamma": ((d * xh).sum((0, 1)), (d.abs() * (eh + n * xh.abs())).sum((0, 1))),
           "dbeta": (d.sum((0, 1)), n * d.abs().sum((0, 1)))}
    return res


def check(name, got, ref, t=None):
    want, bound = ref[name]
    tiny = 2.0 ** -25 if t == torch.float16 else 0.0
    over = (got.double() - want).abs() - bound - tiny
    assert got.shape == want.shape
    assert torch.isfinite(got).all() and (over.numel() == 0 or over.max() <= 0), \
        f"{name}: {(got.double() - want).abs().max():.3e}, {over.max():.3e} over the bound"


def run_and_check(gsv, x, layout, lengths=None):
    t = x["x"].dtype
    ref = reference(x, layout, lengths)
    out, mean, rstd = gsv.add_norm(x["x"], x["y"], x["gamma"], x["beta"], lengths=lengths, layout=layout)
    check("out", out, ref, t)
    check("mean", mean, ref)
    check("rstd", rstd, ref)
    dx, dg, db = gsv.add_norm_backward(x["d_out"], x["x"], x["y"], x["gamma"], mean, rstd, lengths=lengths,
                                       layout=layout)
    check("dx", dx, ref, t)
    check("dgamma", dg, ref)
    check("dbeta", db, ref)
    return out, dx


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("layout,C", [("bct", c) for c in (1, 5, 63, 64, 65, 192, 193, 256, 257, 512, 700, 1025, 2048)]
                         + [("btc", c) for c in (1, 7, 192, 256, 260, 512, 515, 1024, 1030, 2048, 4096, 4097, 8192)])
def test_channels(gsv, dtype, layout, C):
    run_and_check(gsv, make(dtype, layout, 2, C, 45), layout)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("layout", ["bct", "btc"])
@pytest.mark.parametrize("B,T", [(1, 1), (1, 31), (1, 32), (3, 33), (64, 70), (2, 2000)])
def test_frames(gsv, dtype, layout, B, T):
    run_and_check(gsv, make(dtype, layout, B, 192, T, y=False), layout)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("layout", ["bct", "btc"])
@pytest.mark.parametrize("C", [192, 600])
def test_lengths_leave_frames_out(gsv, dtype, layout, C):
    x = make(dtype, layout, 5, C, 77)
    n = torch.tensor([77, 0, 1, 33, 64], dtype=torch.int32, device="cuda")
    frames = (lambda t, b, m: t[b, :, m:]) if layout == "bct" else (lambda t, b, m: t[b, m:])
    for b, m in enumerate(n.tolist()):
        for name in ("x", "y", "d_out"):
            frames(x[name], b, m).fill_(float("nan"))
    ref_in = {k: (torch.nan_to_num(v) if k in ("x", "y", "d_out") else v) for k, v in x.items()}
    ref = reference(ref_in, layout, n)
    out, mean, rstd = gsv.add_norm(x["x"], x["y"], x["gamma"], x["beta"], lengths=n, layout=layout)
    dx, dg, db = gsv.add_norm_backward(x["d_out"], x["x"], x["y"], x["gamma"], mean, rstd, lengths=n, layout=layout)
    for name, got in (("out", out), ("mean", mean), ("rstd", rstd), ("dx", dx), ("dgamma", dg), ("dbeta", db)):
        check(name, got, ref, got.dtype)
    for b, m in enumerate(n.tolist()):
        assert torch.all(frames(out, b, m) == 0) and torch.all(frames(dx, b, m) == 0)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("layout", ["bct", "btc"])
def test_strides_and_alignment(gsv, dtype, layout):
    x = make(dtype, layout, 3, 96, 50)
    g = torch.Generator(device="cuda").manual_seed(4)
    for name, pad in (("x", 1), ("y", 3), ("d_out", 5)):
        s = x[name].shape
        wide = torch.randn(s[0], s[1] + 2, s[2] + pad, generator=g, device="cuda").to(x["x"].dtype)
        x[name] = wide[:, 1:-1, pad:]
    run_and_check(gsv, x, layout)
    x["y"] = x["y"][:1].expand(3, -1, -1)
    run_and_check(gsv, x, layout)


def test_a_large_mean_does_not_cancel(gsv):
    # s = 1000 + noise: a one-pass E[s^2] - E[s]^2 in fp32 would lose the variance.
    for layout in ("bct", "btc"):
        x = make("fp32", layout, 2, 192, 64)
        x["x"] += 1000
        run_and_check(gsv, x, layout)


@pytest.mark.parametrize("layout", ["bct", "btc"])
def test_no_frames(gsv, layout):
    x = make("fp32", layout, 2, 48, 0)
    out, mean, rstd = gsv.add_norm(x["x"], x["y"], x["gamma"], x["beta"], layout=layout)
    assert out.numel() == 0
    dx, dg, db = gsv.add_norm_backward(x["d_out"], x["x"], x["y"], x["gamma"], mean, rstd, layout=layout)
    assert dx.numel() == 0 and torch.all(dg == 0) and torch.all(db == 0)


@pytest.mark.parametrize("layout", ["bct", "btc"])
def test_bits_repeat_and_capture(gsv, layout):
    x = make("bf16", layout, 7, 700, 211)

    def step():
        out, mean, rstd = gsv.add_norm(x["x"], x["y"], x["gamma"], x["beta"], layout=layout)
        return (out, mean, rstd) + gsv.add_norm_backward(x["d_out"], x["x"], x["y"], x["gamma"], mean, rstd,
                                                         layout=layout)

    want = [t.clone() for t in step()]
    for a, b in zip(want, step()):
        assert torch.equal(a, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    x["x"].mul_(2)
    graph.replay()
    got = [t.clone() for t in held]
    for a, b in zip(step(), got):
        assert torch.equal(a, b)


def test_same_results_as_the_handle(gsv):
    # The handle's norm_layers_1 and the stand-alone forward compute the same LayerNorm; each is
    # within its own rounding of the formula.
    sd = gsv.synth.make_state_dict(0)
    sd.update(gsv.synth.make_encp_state_dict())
    dec = gsv.Decoder.load(sd, mode="fp32")
    x = make("fp32", "bct", 2, 192, 40)
    pfx = "enc_p.encoder_ssl.norm_layers_1.0."
    x["gamma"] = torch.as_tensor(sd[pfx + "gamma"]).float().cuda()
    x["beta"] = torch.as_tensor(sd[pfx + "beta"]).float().cuda()
    want = dec.encp_add_norm_device("encoder_ssl", 0, x["x"], x["y"])
    ref = reference(x, "bct", None)
    got = gsv.add_norm(x["x"], x["y"], x["gamma"], x["beta"])[0]
    check("out", want, ref)
    check("out", got, ref)
    dec.close()


def test_refusals(gsv):
    x = make("fp32", "bct", 2, 16, 9)
    with pytest.raises(ValueError):
        gsv.add_norm(x["x"], x["y"][:1], x["gamma"], x["beta"])
    with pytest.raises(ValueError):
        gsv.add_norm(x["x"], None, x["gamma"].half(), x["beta"])
    with pytest.raises(ValueError):
        gsv.add_norm(x["x"], None, x["gamma"], x["beta"], layout="tbc")
    with pytest.raises(ValueError):
        gsv.add_norm(x["x"].transpose(1, 2), None, torch.ones(9, device="cuda"), torch.ones(9, device="cuda"))
    for layout, shape in (("bct", (1, 2049, 4)), ("btc", (1, 4, 8193))):
        C = 2049 if layout == "bct" else 8193
        w = torch.ones(C, device="cuda")
        with pytest.raises(gsv.GsvDecError) as e:
            gsv.add_norm(torch.zeros(shape, device="cuda"), None, w, w, layout=layout)
        assert e.value.status == "GSV_E_INVALID_ARG"


@pytest.mark.parametrize("dtype,layout,B,C,T", [
    # Rings of 2 .. 8 stages that are filled several times over, with frames left out among the others.
    ("bf16", "btc", 8, 1024, 4096), ("fp16", "btc", 5, 2048, 1700), ("fp32", "btc", 1, 8192, 3000),
    ("fp32", "btc", 3, 4096, 1000), ("fp32", "btc", 4, 192, 12000), ("bf16", "btc", 6, 8, 9000),
    ("fp16", "btc", 3, 515, 4000),
    # Clusters that take several tiles each, by vectors and by single frames.
    ("bf16", "bct", 8, 700, 1600), ("bf16", "bct", 8, 700, 1601), ("fp32", "bct", 4, 2048, 2500),
    ("fp32", "bct", 4, 2048, 2499), ("fp16", "bct", 9, 192, 4002), ("fp32", "bct", 16, 300, 1000)])
def test_many_frames_a_block(gsv, dtype, layout, B, C, T):
    x = make(dtype, layout, B, C, T)
    n = torch.tensor([T, T // 3, 0, T - 1, 1, T, 2 * T // 3, 33, T][:B], dtype=torch.int32, device="cuda") \
        if B < 10 else torch.arange(B, dtype=torch.int32, device="cuda") * T // (B - 1)
    if B == 1:
        n -= 5
    for b, m in enumerate(n.tolist()):
        for name in ("x", "y", "d_out"):
            (x[name][b, :, m:] if layout == "bct" else x[name][b, m:]).fill_(float("nan"))
    run_and_check(gsv, x, layout, n)
    gsv.ops_status()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("layout", ["bct", "btc"])
@pytest.mark.parametrize("C", [192, 515, 600])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_statistics_behind_a_length_are_not_used(gsv, dtype, layout, C, bad):
    x = make(dtype, layout, 4, C, 77)
    n = torch.tensor([77, 0, 1, 33], dtype=torch.int32, device="cuda")
    kw = dict(lengths=n, layout=layout)
    _, mean, rstd = gsv.add_norm(x["x"], x["y"], x["gamma"], x["beta"], **kw)
    want = gsv.add_norm_backward(x["d_out"], x["x"], x["y"], x["gamma"], mean, rstd, **kw)
    for b, m in enumerate(n.tolist()):
        mean[b, m:] = rstd[b, m:] = bad
    for a, b in zip(gsv.add_norm_backward(x["d_out"], x["x"], x["y"], x["gamma"], mean, rstd, **kw), want):
        assert torch.equal(a, b)
