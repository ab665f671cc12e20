"""gsvdec_attention_* and gsvdec_norm_* without a GPU: every bad argument is
refused before a device is touched, and workspace sizes are pure functions of
the sizes."""
from __future__ import annotations

import ctypes

import pytest

FAKE = 0x10000  # never followed: each call below is refused first


@pytest.fixture()
def ops(gsv):
    return gsv.ops, gsv.library()


def attention(ops, **kw):
    a = ops._Attention()
    a.dtype, a.B, a.H, a.Hkv, a.Tq, a.Tk, a.D, a.window, a.causal, a.scale = 2, 2, 4, 2, 8, 9, 32, 1, 0, 0.1
    for n in ("q", "k", "v", "rel_k", "rel_v", "o", "lse", "d_o", "dq", "dk", "dv", "drel_k", "drel_v", "workspace"):
        setattr(a, n, FAKE)
    a.workspace_bytes = 1 << 30
    for n in ("q", "o", "d_o", "dq"):
        getattr(a, n + "_stride")[:] = (8 * 4 * 32, 32, 4 * 32)
    for n in ("k", "v", "dk", "dv"):
        getattr(a, n + "_stride")[:] = (9 * 2 * 32, 32, 2 * 32)
    for n, v in kw.items():
        if n.endswith("_stride"):
            getattr(a, n)[:] = v
        else:
            setattr(a, n, v)
    return a


def norm(ops, **kw):
    a = ops._Norm()
    a.dtype, a.layout, a.B, a.C, a.T, a.eps = 2, 0, 2, 16, 10, 1e-5
    for n in ("x", "y", "gamma", "beta", "mean", "rstd", "out", "d_out", "dx", "dgamma", "dbeta", "workspace"):
        setattr(a, n, FAKE)
    a.workspace_bytes = 1 << 30
    for n in ("x", "y", "out", "d_out", "dx"):
        getattr(a, n + "_stride")[:] = (160, 10)
    for n, v in kw.items():
        if n.endswith("_stride"):
            getattr(a, n)[:] = v
        else:
            setattr(a, n, v)
    return a


BAD_ATTENTION = [
    (dict(dtype=3), -4), (dict(dtype=-1), -4), (dict(B=0), -1), (dict(B=70000), -1), (dict(H=0), -1),
    (dict(Hkv=3), -1), (dict(Hkv=0), -1), (dict(Tq=-1), -1), (dict(Tk=(1 << 24) + 1), -1), (dict(D=0), -1),
    (dict(D=129), -1), (dict(window=16), -1), (dict(window=-2), -1), (dict(causal=2), -1), (dict(scale=0.0), -1),
    (dict(scale=float("inf")), -1), (dict(scale=float("nan")), -1), (dict(scale=-1.0), -1), (dict(q=None), -1),
    (dict(k=None), -1), (dict(v=None), -1), (dict(o=None), -1), (dict(rel_k=None), -1), (dict(rel_v=None), -1),
    (dict(q_stride=(-1, 32, 128)), -1), (dict(k_stride=(576, 32, -64)), -1),
]
BAD_FORWARD = [(dict(o_stride=(1024, 0, 128)), -1), (dict(o_stride=(1024, 32, 16)), -1),
               (dict(o_stride=(1000, 32, 128)), -1)]
BAD_BACKWARD = [
    (dict(d_o=None), -1), (dict(lse=None), -1), (dict(dq=None), -1), (dict(dk=None), -1), (dict(dv=None), -1),
    (dict(drel_k=None), -1), (dict(drel_v=None), -1), (dict(workspace=None), -1), (dict(workspace_bytes=64), -1),
    (dict(workspace=FAKE + 8), -1), (dict(dk_stride=(0, 32, 64)), -1), (dict(dv_stride=(576, 32, 31)), -1),
    (dict(dq_stride=(1024, 16, 128)), -1),
]


@pytest.mark.parametrize("kw,status", BAD_ATTENTION + BAD_FORWARD)
def test_forward_refuses(ops, kw, status):
    o, lib = ops
    assert lib.gsvdec_attention_forward(ctypes.byref(attention(o, **kw)), 0, None) == status
    assert lib.gsvdec_last_error()


@pytest.mark.parametrize("kw,status", BAD_ATTENTION + BAD_BACKWARD)
def test_backward_refuses(ops, kw, status):
    o, lib = ops
    assert lib.gsvdec_attention_backward(ctypes.byref(attention(o, **kw)), 0, None) == status


BAD_NORM = [
    (dict(dtype=5), -4), (dict(layout=2), -1), (dict(B=0), -1), (dict(T=-1), -1), (dict(C=0), -1), (dict(C=2049), -1),
    (dict(C=8193, layout=1), -1), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1), (dict(x=None), -1),
    (dict(gamma=None), -1), (dict(mean=None), -1), (dict(rstd=None), -1), (dict(x_stride=(-1, 10)), -1),
]


@pytest.mark.parametrize("kw,status", BAD_NORM + [(dict(beta=None), -1), (dict(out=None), -1),
                                                  (dict(out_stride=(160, 9)), -1), (dict(out_stride=(0, 10)), -1),
                                                  (dict(out_stride=(150, 10)), -1)])
def test_norm_forward_refuses(ops, kw, status):
    o, lib = ops
    assert lib.gsvdec_norm_forward(ctypes.byref(norm(o, **kw)), 0, None) == status


@pytest.mark.parametrize("kw,status", BAD_NORM + [(dict(d_out=None), -1), (dict(dx=None), -1), (dict(dgamma=None), -1),
                                                  (dict(dbeta=None), -1), (dict(workspace=None), -1),
                                                  (dict(workspace_bytes=8), -1), (dict(dx_stride=(160, 0)), -1)])
def test_norm_backward_refuses(ops, kw, status):
    o, lib = ops
    assert lib.gsvdec_norm_backward(ctypes.byref(norm(o, **kw)), 0, None) == status


def test_null_arguments_and_no_such_device(ops):
    o, lib = ops
    n = ctypes.c_size_t()
    assert lib.gsvdec_attention_forward(None, 0, None) == -1
    assert lib.gsvdec_attention_workspace(ctypes.byref(attention(o)), 1, None) == -1
    assert lib.gsvdec_attention_workspace(None, 1, ctypes.byref(n)) == -1
    assert lib.gsvdec_norm_workspace(None, ctypes.byref(n)) == -1
    assert lib.gsvdec_attention_forward(ctypes.byref(attention(o)), 4096, None) == -1
    assert "4096" in lib.gsvdec_last_error().decode()
    assert lib.gsvdec_norm_forward(ctypes.byref(norm(o)), -1, None) == -1


def test_workspace_sizes(ops):
    o, lib = ops
    n = ctypes.c_size_t()
    for T in (0, 1, 64, 5000, 1 << 24):
        a = attention(o, Tq=T, B=65535 if T == 1 << 24 else 2, H=64, Hkv=64, window=15)
        assert lib.gsvdec_attention_workspace(ctypes.byref(a), 1, ctypes.byref(n)) == 0
        assert n.value >= 4 * a.B * a.H * T * 2  # 64-bit arithmetic at the largest sizes
        assert lib.gsvdec_norm_workspace(ctypes.byref(norm(o, T=min(T, 1 << 20))), ctypes.byref(n)) == 0
        assert n.value >= 2 * 16 * 4


def test_more_heads_than_a_launch_has_blocks_are_refused(ops):
    o, lib = ops
    a = attention(o, B=65535, H=512, Hkv=512)
    n = ctypes.c_size_t()
    assert lib.gsvdec_attention_forward(ctypes.byref(a), 0, None) == -1
    assert lib.gsvdec_attention_backward(ctypes.byref(a), 0, None) == -1
    assert lib.gsvdec_attention_workspace(ctypes.byref(a), 1, ctypes.byref(n)) == -1


def test_the_attention_wait_self_test_is_checked(ops):
    _, lib = ops
    assert lib.gsvdec_selftest_attention_wait(None, 0, 10, None) == -1
    assert "limit_ns" in lib.gsvdec_last_error().decode()
    assert lib.gsvdec_selftest_attention_wait(None, 4096, 1000000, None) == -1
    assert "4096" in lib.gsvdec_last_error().decode()


@pytest.mark.parametrize("dtype,off", [(0, 1), (0, 2), (1, 1), (2, 1)])
@pytest.mark.parametrize("name", ["q", "k", "v", "rel_k", "rel_v", "o", "d_o", "dq", "dk", "dv", "drel_k", "drel_v"])
def test_tensors_that_start_inside_an_element_are_refused(ops, dtype, off, name):
    # Device 4096: nothing is launched even where the address is not looked at.
    o, lib = ops
    a = attention(o, dtype=dtype, **{name: FAKE + off})
    call = lib.gsvdec_attention_backward if name.startswith("d") else lib.gsvdec_attention_forward
    assert call(ctypes.byref(a), 4096, None) == -1
    assert "aligned" in lib.gsvdec_last_error().decode()


@pytest.mark.parametrize("name", ["lse", "q_lengths", "k_lengths"])
def test_attention_values_that_start_inside_an_element_are_refused(ops, name):
    o, lib = ops
    for call in (lib.gsvdec_attention_forward, lib.gsvdec_attention_backward):
        assert call(ctypes.byref(attention(o, **{name: FAKE + 2})), 4096, None) == -1
        assert "aligned" in lib.gsvdec_last_error().decode()


@pytest.mark.parametrize("name,off", [("x", 1), ("y", 1), ("out", 1), ("d_out", 1), ("dx", 1), ("gamma", 2),
                                      ("beta", 2), ("mean", 2), ("rstd", 2), ("lengths", 2), ("dgamma", 2),
                                      ("dbeta", 2)])
def test_norm_tensors_that_start_inside_an_element_are_refused(ops, name, off):
    o, lib = ops
    call = lib.gsvdec_norm_backward if name.startswith("d") else lib.gsvdec_norm_forward
    assert call(ctypes.byref(norm(o, **{name: FAKE + off})), 4096, None) == -1
    assert "aligned" in lib.gsvdec_last_error().decode()


def test_aligned_arguments_reach_the_device(ops):
    o, lib = ops
    for dtype, off in ((0, 4), (1, 2), (2, 2)):
        odd = {n: FAKE + off for n in ("q", "k", "v", "rel_k", "rel_v", "o", "d_o", "dq", "dk", "dv", "drel_k", "drel_v")}
        a = attention(o, dtype=dtype, lse=FAKE + 4, q_lengths=FAKE + 4, k_lengths=FAKE + 4, **odd)
        for call in (lib.gsvdec_attention_forward, lib.gsvdec_attention_backward):
            assert call(ctypes.byref(a), 4096, None) == -1
            assert "4096" in lib.gsvdec_last_error().decode()
    for call in (lib.gsvdec_norm_forward, lib.gsvdec_norm_backward):
        assert call(ctypes.byref(norm(o, x=FAKE + 2, d_out=FAKE + 2, gamma=FAKE + 4, mean=FAKE + 4)), 4096, None) == -1
        assert "4096" in lib.gsvdec_last_error().decode()
