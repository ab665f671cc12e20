"""Operators called by several host threads at once, each on its own stream and
with its own tensors.  A launch needs its kernel's shared-memory limit to be at
least its own size, whatever the other threads' calls need.  The threads call
the C functions with arguments packed beforehand, so that they spend their time
there (and not waiting for the interpreter)."""
from __future__ import annotations

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def recorded(monkeypatch, gsv, call):
    """The C calls that call() makes: [(function, packed arguments, device)], with its results."""
    made, c = [], gsv.ops._get()
    with monkeypatch.context() as m:
        for name in ("attention_forward", "attention_backward", "norm_forward", "norm_backward"):
            def record(a, index, stream, f=getattr(c, name)):
                made.append((f, a, index))
                return f(a, index, stream)

            m.setattr(c, name, record)
        kept = call()
    torch.cuda.synchronize()
    return made, kept


def together(jobs, turns):
    """Each of jobs (lists of recorded calls) `turns` times over, in a thread of its own; the errors seen."""
    errors, start = [], threading.Barrier(len(jobs))
    streams = [torch.cuda.Stream() for _ in jobs]

    def work(calls, stream):
        start.wait()
        for _ in range(turns):
            for f, a, index in calls:
                rc = f(a, index, stream)
                if rc:
                    errors.append(rc)
                    return

    threads = [threading.Thread(target=work, args=(j, s.cuda_stream)) for j, s in zip(jobs, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return errors


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_with_and_without_a_window(gsv, monkeypatch, dtype, D):
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(1, 1, 9, D, generator=g, device="cuda").to(dtype) for _ in range(3))
    rel = [(torch.randn(31, D, generator=g, device="cuda") * 0.1).to(dtype) for _ in range(2)]
    jobs, kept = [], []
    for kw in (dict(rel_k=rel[0], rel_v=rel[1]), {}) * 2:
        made, out = recorded(monkeypatch, gsv, lambda: gsv.attention(q, k, v, **kw))
        jobs.append(made)
        kept.append((out, [t.clone() for t in out]))
    assert together(jobs, 10000) == []
    for out, want in kept:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_norms_of_other_widths_after_every_kernel_was_used(gsv, monkeypatch):
    # All kernels of the [B, T, C] norm (3 types, aligned or single elements, 6 shares of a row, both directions),
    # then pairs of widths that one of them serves.
    shares = [(256, 24), (512, 264), (1024, 520), (2048, 1032), (4096, 2056), (8192, 4104)]

    def step(x, w):
        out, mean, rstd = gsv.add_norm(x, x, w, w, layout="btc")
        return (out, mean, rstd) + gsv.add_norm_backward(x, x, x, w, mean, rstd, layout="btc"), x, w

    pairs = []
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        for off in (1, 0):
            for widths in shares:
                pair = []
                for C in widths:
                    x, w = torch.randn(1, 9, C + off, device="cuda").to(dtype)[..., off:], torch.randn(C, device="cuda")
                    made, kept = recorded(monkeypatch, gsv, lambda: step(x, w))
                    # The backward's workspace was torch's to give away when the call returned.
                    ws = torch.empty(gsv.ops._norm_workspace(*gsv.ops._norm_in(gsv.ops._get(), x, x, None, "btc")[0]),
                                     dtype=torch.uint8, device="cuda")
                    f, a, index = made[1]
                    made[1] = (f, a[:-16] + ws.data_ptr().to_bytes(8, "little") + a[-8:], index)
                    pair.append((made, kept, ws, [t.clone() for t in kept[0]]))
                pairs.append(pair)
    for pair in pairs:
        assert together([p[0] for p in pair], 2000) == []
        for _, kept, _, want in pair:
            assert all(torch.equal(a, b) for a, b in zip(kept[0], want))


def test_calls_on_several_streams_at_once(gsv):
    # Kernels that share SMs, their shared memory and TMEM: every call has the bits it has alone.
    g = torch.Generator(device="cuda").manual_seed(0)

    def rows(dtype, *shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    def attention(q, k, v, do, **kw):
        o, lse = gsv.attention(q, k, v, **kw)
        return (o, lse) + gsv.attention_backward(do, q, k, v, o, lse, **kw)[:3]

    def norm(x, w):
        out, mean, rstd = gsv.add_norm(x, x, w, w, layout="btc")
        return (out, mean, rstd) + gsv.add_norm_backward(x, x, x, w, mean, rstd, layout="btc")

    bf, half, f32 = torch.bfloat16, torch.float16, torch.float32
    a = [rows(bf, 1, 8, n, 64) for n in (128, 4096, 4096, 128)]  # key tiles split over clusters
    b = [rows(bf, 4, 2, 500, 96) for _ in range(4)]
    c = [rows(half, 2, 4, 300, 32) for _ in range(4)]
    d = [rows(f32, 2, 2, 200, 128) for _ in range(4)]
    x, w = rows(bf, 4, 1024, 512), rows(f32, 512)
    jobs = [lambda: attention(*a), lambda: attention(*b), lambda: attention(*c, causal=True), lambda: attention(*d),
            lambda: norm(x, w)]
    want = [[t.clone() for t in j()] for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(30):
        outs = []
        for s, j in zip(streams, jobs):
            with torch.cuda.stream(s):
                outs.append(j())
        torch.cuda.synchronize()
        for out, ref in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(out, ref))
    gsv.ops_status()
