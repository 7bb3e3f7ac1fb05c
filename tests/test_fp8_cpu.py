"""What the 8-bit operators refuse, checked before anything reaches a device, and their plain forms against the definitions."""

from __future__ import annotations

import pytest
import torch

import plain_fp8 as pf
from acvram_b200.kernels import ops
from acvram_b200.kernels.ops import FP8, KernelError


def pair(R, C, block_rows=1):
    q, s = ops.fp8_rows(R, C, "cpu")
    return q, (s if block_rows == 1 else torch.empty((pf.groups(R), pf.groups(C))))


def refused(words, call, *args, **kw):
    with pytest.raises(KernelError, match=words):
        call(*args, **kw)


def test_fp8_rows_gives_aligned_rows():
    for R, C in ((1, 1), (3, 100), (5, 128), (0, 16)):
        q, s = ops.fp8_rows(R, C, "cpu")
        assert q.shape == (R, C) and q.dtype == FP8 and (q.stride(0) % 16 == 0) and s.shape == (R, pf.groups(C))


def test_quantize_refuses():
    x = torch.zeros((4, 200))
    q, s = pair(4, 200)
    refused("CPU tensor", ops.quantize_fp8, x, q, s)
    refused("x must be", ops.quantize_fp8, x.half(), q, s)
    refused("x must be", ops.quantize_fp8, torch.zeros((200, 4)).t(), q, s)
    refused("the result must be", ops.quantize_fp8, x, q.view(torch.uint8), s)
    refused("the result must be", ops.quantize_fp8, x, q[:, :128], s)
    refused("scales of the result", ops.quantize_fp8, x, q, s[:, :1])
    refused("scales of the result", ops.quantize_fp8, x, q, s, 128)
    refused("scales of the result", ops.quantize_fp8, x, q, s.double())
    refused("block_rows", ops.quantize_fp8, x, q, s, 64)
    refused("a matrix", ops.quantize_fp8, x[0], q, s)


def test_linear_refuses():
    x, xs = pair(4, 256)
    w, ws = pair(300, 256, 128)
    out = torch.empty((4, 300))
    refused("CPU tensor", ops.linear_fp8, x, xs, w, ws, out)
    refused("w must be", ops.linear_fp8, x[:, :128], xs[:, :1], w, ws, out)
    refused("scales of x", ops.linear_fp8, x, xs[:, :1], w, ws, out)
    refused("scales of w", ops.linear_fp8, x, xs, w, ws[:2], out)
    refused("out must be", ops.linear_fp8, x, xs, w, ws, out.half())
    refused("out must be", ops.linear_fp8, x, xs, w, ws, out[:, :299])
    refused("out must be", ops.linear_fp8, x, xs, w, ws, torch.empty((300, 4)).t())
    refused("x must be", ops.linear_fp8, x.view(torch.int8), xs, w, ws, out)


def test_gated_linear_refuses():
    x, xs = pair(4, 256)
    g, gs = pair(200, 256, 128)
    q, s = pair(4, 200)
    refused("CPU tensor", ops.linear_fp8_swiglu, x, xs, g, gs, g, gs, q, s)
    refused("up must be", ops.linear_fp8_swiglu, x, xs, g, gs, g[:100], gs[:1], q, s)
    refused("scales of up", ops.linear_fp8_swiglu, x, xs, g, gs, g, gs[:1], q, s)
    refused("the result must be", ops.linear_fp8_swiglu, x, xs, g, gs, g, gs, torch.empty((4, 200)), s)
    refused("scales of the result", ops.linear_fp8_swiglu, x, xs, g, gs, g, gs, q, s[:, :1])


def test_norms_refuse():
    x, d, w = torch.zeros((4, 256)), torch.zeros((4, 256), dtype=torch.bfloat16), torch.zeros(256)
    q, s = pair(4, 256)
    refused("CPU tensor", ops.add_gated_norms, x, d, q, s, weight=w)
    refused("wants a weight", ops.add_gated_norms, x, d, q, s)
    refused("no delta", ops.add_gated_norms, x, None, q, s, weight=w, post_weight=w)
    refused("no delta", ops.add_gated_norms, x, None, q, s, weight=w, gate=w)
    refused("without a result", ops.add_gated_norms, x, d, None, s)
    refused("out_scales go with", ops.add_gated_norms, x, d, q, None, weight=w)
    refused("out_scales go with", ops.add_gated_norms, x, d, x.clone(), s, weight=w)
    refused("delta must be", ops.add_gated_norms, x, d[:3], q, s, weight=w)
    refused("x must be", ops.add_gated_norms, x.half(), d, q, s, weight=w)
    refused("gate by tokens", ops.add_gated_norms, x, d, q, s, weight=w, gate=torch.zeros((4, 128)))
    refused("gate by channels", ops.add_gated_norms, x, d, q, s, weight=w, gate=torch.zeros(255))
    refused("gate by channels", ops.add_gated_norms, x, d, q, s, weight=w, gate=w.bfloat16())
    refused("weight must be", ops.add_gated_norms, x, d, q, s, weight=torch.zeros(512)[::2])
    refused("post_weight must be", ops.add_gated_norms, x, d, q, s, weight=w, post_weight=w.double())


def test_records_are_as_long_as_the_structs():
    """Pointers, then 64-bit strides, then 32-bit fields: no padding in front of any of them, so the packed length is their sum."""
    assert ops._LINEAR_ARGS.size == 10 * 8 + 8 * 8 + 7 * 4
    assert ops._QUANTIZE_ARGS.size == 4 * 8 + 3 * 8 + 5 * 4
    assert ops._NORMS_ARGS.size == 9 * 8 + 5 * 8 + 8 * 4 + 3 * 4


def test_plain_quantisation_is_near_what_it_stands_for():
    x = torch.randn((200, 300), generator=torch.Generator().manual_seed(1))
    for block_rows in (1, 128):
        q, s = pf.quantize(x, block_rows)
        off = (pf.values(q, s, block_rows) - x.double()).abs()
        assert bool((off <= x.double().abs() * 2.0 ** -4 * (1 + 1e-6) + pf.spread(s.double(), 200, 300, block_rows) * 2.0 ** -10).all())


# ----------------------------------------------------------------------------- configurations and weight files
def fp8_config(**quant):
    from conftest import tiny_config
    cfg = tiny_config("F").to_dict()
    cfg["quantization_config"] = {"quant_method": "fp8", "fmt": "e4m3", "activation_scheme": "dynamic", "weight_block_size": [128, 128], **quant}
    return cfg


def test_configuration_of_8_bit_weights():
    from acvram_b200.config import ConfigError, Qwen3Config
    from conftest import tiny_config
    cfg = Qwen3Config.from_dict(fp8_config())
    assert cfg.weights_fp8 and Qwen3Config.from_dict(cfg.to_dict()) == cfg
    assert "quantization_config" not in tiny_config("F").to_dict() and "weights_fp8" not in tiny_config("F").to_dict()
    assert not Qwen3Config.from_dict(fp8_config(quant_method="other")).weights_fp8
    for patch in ({"weight_block_size": [64, 128]}, {"weight_block_size": None}, {"activation_scheme": "static"}, {"fmt": "e5m2"}):
        with pytest.raises(ConfigError, match="quantization_config"):
            Qwen3Config.from_dict(fp8_config(**patch))


def test_weights_in_8_bits_are_asked_of_the_configuration():
    from acvram_b200.config import ConfigError
    from acvram_b200.models import needs_of_plan, with_weights
    from acvram_b200.config import family_of
    from conftest import tiny_config
    cfg = with_weights(tiny_config("F"), "fp8")
    needs = needs_of_plan(family_of(cfg.to_dict()).build_plan(cfg))
    assert needs["model.layers.0.mlp.down_proj.weight"].role == "fp8"
    scale = needs["model.layers.1.self_attn.q_proj.weight_scale_inv"]
    assert scale.shape == (4, 2) and scale.optional
    assert needs["model.embed_tokens.weight"].role == "embedding" and "lm_head.weight_scale_inv" not in needs
    assert with_weights(cfg, None) is cfg
    with pytest.raises(ConfigError, match="built"):
        with_weights(cfg, "int4")
    with pytest.raises(ConfigError, match="not built for"):
        with_weights(type("C", (), {"architecture": "Other"})(), "fp8")


def test_a_weight_file_with_half_of_a_quantised_matrix():
    from acvram_b200.parts.linear import Fp8Linear
    from acvram_b200.weights.needs import WeightError
    q = torch.zeros((128, 128)).to(FP8)
    with pytest.raises(WeightError, match="w_scale_inv"):
        Fp8Linear.matrix({"w": q}, "w", "cpu")
    with pytest.raises(WeightError, match="beside block scales"):
        Fp8Linear.matrix({"w": q.float(), "w_scale_inv": torch.ones((1, 1))}, "w", "cpu")


def test_loader_keeps_e4m3_where_it_is_asked_for(tmp_path):
    from safetensors.torch import save_file
    from acvram_b200.weights import load_tensors
    from acvram_b200.weights.needs import TensorNeed, WeightError
    save_file({"w": torch.ones((4, 8)).to(FP8)}, str(tmp_path / "model.safetensors"))
    assert load_tensors(tmp_path, {"w": TensorNeed((4, 8), "fp8")})["w"].dtype == FP8
    with pytest.raises(WeightError, match="unsupported dtype"):
        load_tensors(tmp_path, {"w": TensorNeed((4, 8))})


def test_parts_refuse_what_is_not_built_beside_8_bit_weights():
    from acvram_b200.parts.feed_forward import SwiGLU
    from acvram_b200.parts.mixers import Attention
    from acvram_b200.parts.plan import PartSpec
    with pytest.raises(ValueError, match="8-bit"):
        SwiGLU(64, 128, activation="gelu_tanh", fp8=True)
    with pytest.raises(ValueError, match="8-bit"):
        Attention(64, 4, 2, 16, PartSpec("none", {}), bias=True, fp8=True)


def test_command_line_has_the_choice():
    from acvram_b200.cli import build_parser
    args = build_parser().parse_args(["generate", "folder", "--weights", "fp8"])
    assert args.weights == "fp8"
    assert build_parser().parse_args(["bench", "folder"]).weights is None


def test_a_bias_beside_8_bit_weights_is_refused():
    """Weights in more bits are served with the biases that a file happens to hold; here they must not be left out in silence."""
    from acvram_b200.parts.linear import Fp8Linear
    from acvram_b200.weights.needs import WeightError
    needs = Fp8Linear.needs("q_proj.weight", 256, 128)
    assert needs["q_proj.bias"].optional and needs["q_proj.bias"].shape == (256,)
    with pytest.raises(WeightError, match="q_proj.bias .*without biases"):
        Fp8Linear.matrix({"q_proj.weight": torch.zeros((128, 128)).to(FP8), "q_proj.weight_scale_inv": torch.ones((1, 1)),
                          "q_proj.bias": torch.ones(128)}, "q_proj.weight", "cpu")
