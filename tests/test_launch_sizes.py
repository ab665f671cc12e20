"""The number of blocks of the attention's launches (csrc/attn_launch.h), at
sizes that need more than 32 bits on the way, and the refusal of calls that
need more blocks than a launch has."""
from __future__ import annotations

import ctypes
import subprocess

import pytest

from conftest import ROOT
from test_ops_abi import attention, ops  # noqa: F401

HARNESS = r"""
#include "attn_launch.h"

#include <cstdio>
#include <cstdlib>

int main(int, char** v) {
  gsv::AttnArgs a{};
  a.ty = (gsv::Ty)std::atoi(v[1]);
  a.B = std::atoi(v[2]), a.H = std::atoi(v[3]), a.Hkv = std::atoi(v[4]);
  a.Tq = std::atoi(v[5]), a.Tk = std::atoi(v[6]), a.D = std::atoi(v[7]);
  const gsv::RowBlocks r = gsv::row_blocks(a);
  std::printf("%lld %lld %lld %lld\n", (long long)r.q, (long long)r.k, (long long)gsv::attn_most_blocks(a, false),
              (long long)gsv::attn_most_blocks(a, true));
  return 0;
}
"""


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    d = tmp_path_factory.mktemp("blocks")
    (d / "h.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-I", str(ROOT / "gpt-sovits-rs_b200" / "csrc"), "-I",
                    "/usr/local/cuda/include", str(d / "h.cpp"), "-o", str(d / "h")], check=True)
    return d / "h"


def blocks(harness, *args):
    out = subprocess.run([str(harness), *map(str, args)], check=True, capture_output=True, text=True).stdout
    return list(map(int, out.split()))


def up(n, m):
    return -(-n // m)


@pytest.mark.parametrize("ty", [0, 1, 2])
@pytest.mark.parametrize("B,H,Hkv,Tq,Tk,D", [
    (1, 1, 1, 1, 1, 1), (2, 4, 2, 200, 61, 64), (3, 6, 3, 129, 128, 96), (16, 2, 2, 500, 500, 96),
    # One key head of many queries' heads over long keys: key rows are counted by key heads.
    (1, 65535, 1, 1, 1 << 24, 32), (1, 65535, 1, 1, 1 << 24, 128), (65535, 256, 1, 8, 4096, 64),
    (65535, 256, 256, 1 << 24, 1 << 24, 128), (1, 1, 1, 0, 77, 20), (1, 1, 1, 77, 0, 20)])
def test_blocks(harness, ty, B, H, Hkv, Tq, Tk, D):
    rows = {True: 128, False: 64 if D <= 64 else 32}[D <= 32]
    tile = 64 if ty == 0 else 128
    q = up(up(Tq, 128) * 128, rows) * H * B
    k = up(Tk, rows) * Hkv * B if ty == 1 else 0
    fwd = up(Tq, tile) * H * B
    bwd = max(q + k, fwd + up(Tk, tile) * Hkv * B)
    assert blocks(harness, ty, B, H, Hkv, Tq, Tk, D) == [q, k, fwd, bwd]


def test_more_tiles_than_a_launch_has_blocks_are_refused(ops):  # noqa: F811
    o, lib = ops
    big = attention(o, dtype=1, B=65535, H=256, Hkv=256, Tq=1 << 24, Tk=1 << 24, D=1, window=-1,
                    **{n + "_stride": (1 << 39, 1 << 30, 1) for n in ("o", "dq", "dk", "dv")})
    big.workspace_bytes = 1 << 60
    for call in (lib.gsvdec_attention_forward, lib.gsvdec_attention_backward):
        assert call(ctypes.byref(big), 4096, None) == -1
        assert "blocks" in lib.gsvdec_last_error().decode()
    # Many heads on one key head over long keys fit a launch.
    wide = attention(o, dtype=1, B=1, H=65535, Hkv=1, Tq=1, Tk=1 << 24, D=1, window=-1,
                     **{n + "_stride": (1 << 30, 1, 1) for n in ("o", "dq", "dk", "dv")})
    wide.workspace_bytes = 1 << 60
    for call in (lib.gsvdec_attention_forward, lib.gsvdec_attention_backward):
        assert call(ctypes.byref(wide), 4096, None) == -1
        assert "4096" in lib.gsvdec_last_error().decode()
