"""gsvdec_encp_attention (the text encoder's self-attention from its weights)
against the formulas in 64 bits, alone and as the `attn` of gsvdec_encp_layer."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle
from attn_ref import reference
from conftest import rel_max, snr_db

pytestmark = pytest.mark.gpu

LAYERS = {"encoder_ssl": 1, "encoder_text": 2}
FP32_REL, BF16_SNR_DB = 1e-4, 30.0  # the bars of the other enc_p chains


@pytest.fixture(scope="module")
def sd(gsv):
    sd = gsv.synth.make_state_dict(0, init="unit", bias="rand")
    sd.update(gsv.synth.make_encp_state_dict(layers=LAYERS))
    sd.update(gsv.synth.make_encp_attention_state_dict(layers=LAYERS))
    return sd


@pytest.fixture(scope="module")
def handles(gsv, sd):
    hs = {m: gsv.Decoder.load(sd, device=0, mode=m) for m in ("fp32", "bf16", "fp32tc")}
    yield hs
    for h in hs.values():
        h.close()


def expected(sd, stack, layer, x, lengths):
    p = f"enc_p.{stack}.attn_layers.{layer}."
    w = {k[len(p):]: torch.as_tensor(v).double() for k, v in sd.items() if k.startswith(p)}
    x = torch.as_tensor(x).double()
    B, C, T = x.shape
    D = w["emb_rel_k"].shape[-1]

    def heads(name):
        y = torch.einsum("oi,bit->bto", w[name + ".weight"][..., 0], x) + w[name + ".bias"]
        return y.view(B, T, C // D, D).transpose(1, 2)

    n = None if lengths is None else torch.as_tensor(lengths)
    o = reference(heads("conv_q"), heads("conv_k"), heads("conv_v"), q_lengths=n, k_lengths=n,
                  rel_k=w["emb_rel_k"][0], rel_v=w["emb_rel_v"][0])["o"]
    out = torch.einsum("oi,bti->bot", w["conv_o.weight"][..., 0], o.transpose(1, 2).reshape(B, T, C))
    out = out + w["conv_o.bias"].view(1, C, 1)
    if n is not None:
        for b, m in enumerate(lengths):
            out[b, :, m:] = 0
    return out.numpy()


def check(mode, got, want):
    if mode == "bf16":
        assert snr_db(got, want) >= BF16_SNR_DB
    else:
        assert rel_max(got, want) <= FP32_REL


@pytest.mark.parametrize("mode", ["fp32", "bf16", "fp32tc"])
@pytest.mark.parametrize("stack,layer,B,T,lengths", [
    ("encoder_ssl", 0, 1, 1, None), ("encoder_text", 1, 1, 37, None), ("encoder_text", 0, 3, 200, [200, 1, 77]),
    ("encoder_ssl", 0, 2, 333, [0, 333])])
def test_matches_the_formulas(gsv, handles, sd, mode, stack, layer, B, T, lengths):
    x = np.random.default_rng(T).standard_normal((B, 192, T)).astype(np.float32)
    want = expected(sd, stack, layer, x, lengths)
    h = handles[mode]
    check(mode, h.encp_attention(stack, layer, x, lengths), want)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got = h.encp_attention_device(stack, layer, torch.as_tensor(x).cuda(), ln)
    check(mode, got.cpu().numpy(), want)


@pytest.mark.parametrize("mode", ["fp32", "bf16"])
def test_whole_encoder_layer(handles, sd, mode):
    x = np.random.default_rng(3).standard_normal((2, 192, 120)).astype(np.float32)
    lengths = [120, 90]
    x[1, :, 90:] = 0
    attn = expected(sd, "encoder_text", 0, x, lengths).astype(np.float32)
    n1 = "enc_p.encoder_text.norm_layers_1.0."
    h1 = oracle.layer_norm(x, sd[n1 + "gamma"], sd[n1 + "beta"], y=attn)
    want = oracle.encp_ffn(sd, "encoder_text", 0, h1, lengths)
    hd = handles[mode]
    got = hd.encp_layer("encoder_text", 0, x, hd.encp_attention("encoder_text", 0, x, lengths), lengths)
    check(mode, got, want)
    assert np.all(got[1, :, 90:] == 0)


def test_from_a_file(gsv, sd, tmp_path, handles):
    from safetensors.numpy import save_file
    path = tmp_path / "m.safetensors"
    save_file({k: np.ascontiguousarray(v) for k, v in sd.items()}, str(path))
    h = gsv.Decoder.load_file(str(path), mode="bf16")
    x = np.random.default_rng(5).standard_normal((1, 192, 50)).astype(np.float32)
    assert np.array_equal(h.encp_attention("encoder_text", 1, x), handles["bf16"].encp_attention("encoder_text", 1, x))
    h.close()


def test_refusals(gsv, sd, handles):
    x = np.zeros((1, 192, 4), np.float32)
    for stack, layer in (("encoder2", 0), ("encoder_text", 2), (7, 0)):
        with pytest.raises(gsv.GsvDecError) as e:
            handles["fp32"].encp_attention(stack, layer, x)
        assert e.value.status == "GSV_E_INVALID_ARG"
    part = {k: v for k, v in sd.items() if "encoder_ssl.attn_layers" not in k}
    part["enc_p.encoder_text.attn_layers.0.emb_rel_k"] = np.zeros((1, 40, 96), np.float32)  # even
    h = gsv.Decoder.load(part, mode="fp32")  # loads: the attention is optional
    for stack in ("encoder_ssl", "encoder_text"):
        with pytest.raises(gsv.GsvDecError) as e:
            h.encp_attention(stack, 0, x)
        assert e.value.status == "GSV_E_UNSUPPORTED"
    h.encp_attention("encoder_text", 1, x)
    h.close()
