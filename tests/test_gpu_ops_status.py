"""Where a bounded device wait that gave up is reported: the attention of a
handle's enc_p call on the handle (gsvdec_sync_status, the next call on it), an
operator's by gsvdec_ops_status.  The give-ups are made by
gsvdec_selftest_attention_wait, a wait of 1 ms with nothing else in flight."""
from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dec(gsv):
    sd = gsv.synth.make_state_dict(0)
    layers = {"encoder_ssl": 1}
    sd.update(gsv.synth.make_encp_state_dict(layers=layers))
    sd.update(gsv.synth.make_encp_attention_state_dict(layers=layers))
    d = gsv.Decoder.load(sd, device=0, mode="bf16")
    yield d
    d.close()


@pytest.fixture()
def x():
    return np.random.default_rng(1).standard_normal((2, 192, 40)).astype(np.float32)


def gave_up(gsv, call):
    with pytest.raises(gsv.GsvDecError) as e:
        call()
    assert e.value.status == "GSV_E_TIMEOUT"


def test_the_handle_reports_its_attention(gsv, dec, x):
    gsv.ops_status()
    want = dec.encp_attention("encoder_ssl", 0, x)
    dec.selftest_attention_wait()
    gave_up(gsv, dec.sync_status)
    dec.sync_status()  # reported once
    dec.selftest_attention_wait()
    torch.cuda.synchronize()
    gave_up(gsv, lambda: dec.encp_attention_device("encoder_ssl", 0, torch.as_tensor(x).cuda()))  # at its entry
    dec.selftest_attention_wait()
    gave_up(gsv, lambda: dec.encp_attention("encoder_ssl", 0, x))  # a call on host memory
    gsv.ops_status()  # no operator gave up
    assert np.array_equal(dec.encp_attention("encoder_ssl", 0, x), want)


def test_a_call_on_a_handle_leaves_the_operators_report(gsv, dec, x):
    want = dec.encp_attention("encoder_ssl", 0, x)
    gsv.ops.selftest_wait()
    torch.cuda.synchronize()
    assert np.array_equal(dec.encp_attention("encoder_ssl", 0, x), want)
    dec.sync_status()
    gave_up(gsv, gsv.ops_status)
    gsv.ops_status()


def test_the_limit_is_checked(gsv, dec):
    for call in (gsv.ops.selftest_wait, dec.selftest_attention_wait):
        with pytest.raises(gsv.GsvDecError) as e:
            call(10)
        assert e.value.status == "GSV_E_INVALID_ARG"
    gsv.ops_status()


def test_another_thread_does_not_take_the_report(gsv):
    gsv.ops_status()
    gsv.ops.selftest_wait()
    torch.cuda.synchronize()
    seen = []

    def other():
        try:
            gsv.ops_status()
            seen.append("GSV_OK")
        except gsv.GsvDecError as e:
            seen.append(e.status)

    t = threading.Thread(target=other)
    t.start()
    t.join()
    assert seen == ["GSV_E_TIMEOUT"]  # a thread sees every give-up it has not been told of
    gave_up(gsv, gsv.ops_status)
    gsv.ops_status()
