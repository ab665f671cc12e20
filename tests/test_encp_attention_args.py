"""The tensors of an encp_attention call are checked against the handle before
anything reads them (on the CPU: a stand-in for a handle of 192 channels, whose
device number -1 is the one that torch gives CPU tensors)."""
from __future__ import annotations

import numpy as np
import pytest
import torch


@pytest.fixture()
def dec(gsv):
    d = gsv.Decoder.__new__(gsv.Decoder)
    d._h, d.info, d._encp_channels = None, {"device": -1}, 192
    return d


def refused_by_the_library(gsv, call):
    # The stand-in has no handle: a call whose tensors are accepted ends there.
    with pytest.raises(gsv.GsvDecError) as e:
        call()
    assert e.value.status == "GSV_E_INVALID_ARG" and "handle is NULL" in str(e.value)


def test_host_arrays(gsv, dec):
    refused_by_the_library(gsv, lambda: dec.encp_attention(0, 0, np.zeros((2, 192, 5), np.float32), [5, 3]))
    for x, n in ((np.zeros((2, 100, 5), np.float32), None), (np.zeros((2, 193, 5), np.float32), None),
                 (np.zeros((2, 192, 5), np.float32), [5])):
        with pytest.raises(ValueError):
            dec.encp_attention(0, 0, x, n)


def test_device_tensors(gsv, dec):
    x, n = torch.zeros(2, 192, 5), torch.ones(2, dtype=torch.int32)
    refused_by_the_library(gsv, lambda: dec.encp_attention_device(0, 0, x, n, out=torch.empty_like(x), stream=0))
    bad = [dict(x=torch.zeros(2, 100, 5)), dict(x=x.double()), dict(x=torch.zeros(2, 5, 192).transpose(1, 2)),
           dict(lengths=n.long()), dict(lengths=n[:1]), dict(lengths=torch.ones(4, dtype=torch.int32)[::2]),
           dict(out=torch.empty(2, 192, 4)), dict(out=torch.empty(1, 192, 5)), dict(out=torch.empty_like(x).double()),
           dict(out=torch.empty(2, 5, 192).transpose(1, 2))]
    for kw in bad:
        with pytest.raises(ValueError):
            dec.encp_attention_device(0, 0, kw.get("x", x), kw.get("lengths", n), out=kw.get("out"), stream=0)
    dec.info = {"device": 0}
    with pytest.raises(ValueError):
        dec.encp_attention_device(0, 0, x, n, stream=0)
