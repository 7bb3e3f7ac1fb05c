"""A model's 8-bit matrices, all seven of a layer, are those of its folder, scale for scale."""

from __future__ import annotations

import os

import pytest
import torch
from safetensors.torch import load_file

import plain_fp8 as pf
from test_fp8_model_gpu import engine

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["A", "B", "D", "E", "F"])
def test_every_matrix_of_a_model_is_its_folders(tiny_folders, name):
    tensors = load_file(os.path.join(tiny_folders[name], "model.safetensors"))
    eng = engine(tiny_folders[name], "bfloat16", name, weights="fp8")
    for i, block in enumerate(eng.model.blocks):
        at = f"model.layers.{i}."
        parts = {"qkv": (block.mixer.qkv, ["self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj"]), "o": (block.mixer.o, ["self_attn.o_proj"]),
                 "gate": (block.feed_forward.gate, ["mlp.gate_proj"]), "up": (block.feed_forward.up, ["mlp.up_proj"]),
                 "down": (block.feed_forward.down, ["mlp.down_proj"])}
        for what, (linear, names) in parts.items():
            rows = torch.cat([tensors[f"{at}{n}.weight"].float() for n in names])
            first = 0
            for values, scales in linear.matrices:
                want, want_scales = pf.quantize(rows[first:first + values.shape[0]], 128)
                assert torch.equal(scales.cpu(), want_scales) and torch.equal(values.cpu().view(torch.uint8), want.view(torch.uint8)), (i, what, first)
                first += values.shape[0]
            assert first == rows.shape[0]
