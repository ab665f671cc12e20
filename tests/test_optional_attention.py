"""A checkpoint's enc_p attention is optional: tensors of it in a form that the
library does not take do not keep the file from loading (checked without a
GPU: what the loader reports next is a decoder tensor that is missing)."""
from __future__ import annotations

import json
import struct

import pytest


def write(path, tensors):
    """A safetensors file of zeros: {name: (dtype, shape)}."""
    size = {"F64": 8, "F32": 4, "I64": 8, "F8_E4M3": 1}
    head, at = {}, 0
    for name, (dtype, shape) in tensors.items():
        n = size[dtype]
        for d in shape:
            n *= d
        head[name] = {"dtype": dtype, "shape": list(shape), "data_offsets": [at, at + n]}
        at += n
    text = json.dumps(head).encode()
    path.write_bytes(struct.pack("<Q", len(text)) + text + bytes(at))


@pytest.mark.parametrize("name", ["conv_q.weight", "emb_rel_k", "scale"])
@pytest.mark.parametrize("dtype,shape", [("F64", (1, 9, 96)), ("I64", (4,)), ("F8_E4M3", (4, 4, 1)), ("F32", ()),
                                         ("F32", (1, 1, 1, 2, 2))])
def test_attention_tensors_of_another_form_are_left_out(gsv, tmp_path, name, dtype, shape):
    path = tmp_path / "m.safetensors"
    write(path, {"dec.conv_pre.weight": ("F32", (512, 192, 7)),
                 "enc_p.encoder_text.attn_layers.0." + name: (dtype, shape)})
    with pytest.raises(gsv.GsvDecError) as e:
        gsv.Decoder.load_file(str(path), mode="bf16")
    assert e.value.status == "GSV_E_MISSING_KEY" and "dec." in str(e.value)


def test_other_tensors_of_another_form_are_refused(gsv, tmp_path):
    path = tmp_path / "m.safetensors"
    write(path, {"dec.conv_pre.weight": ("F64", (512, 192, 7))})
    with pytest.raises(gsv.GsvDecError) as e:
        gsv.Decoder.load_file(str(path), mode="bf16")
    assert e.value.status == "GSV_E_DTYPE"
