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
