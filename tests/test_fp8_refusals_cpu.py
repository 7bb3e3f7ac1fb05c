"""What a folder's or a caller's words about 8-bit weights may not silently lose."""

from __future__ import annotations

import pytest


def fp8_config(**quant):
    from conftest import tiny_config
    cfg = tiny_config("F").to_dict()
    cfg["quantization_config"] = {"quant_method": "fp8", "fmt": "e4m3", "activation_scheme": "dynamic", "weight_block_size": [128, 128], **quant}
    return cfg


@pytest.mark.parametrize("key", ["modules_to_not_convert", "ignored_layers"])
@pytest.mark.parametrize("name", [
    "model.layers.0.self_attn.q_proj", "model.layers.1.mlp.down_proj.weight", "model.layers.0", "model.layers.1.self_attn", "mlp", "q_proj",
    "up_proj", "model", "layers.1.mlp.gate_proj", "model.layers.0.mlp.gate", "language_model.model.layers.0.self_attn.o_proj"])
def test_matrices_that_a_folder_keeps_in_more_bits_are_refused(key, name):
    """Such a matrix would be quantised as it is loaded, and the model would not be the folder's."""
    from acvram_b200.config import ConfigError, Qwen3Config
    with pytest.raises(ConfigError, match=f"{key}.*'{name}'"):
        Qwen3Config.from_dict(fp8_config(**{key: ["lm_head", name]}))


@pytest.mark.parametrize("key", ["modules_to_not_convert", "ignored_layers"])
@pytest.mark.parametrize("names", [None, [], ["lm_head"], ["lm_head", "model.embed_tokens", "model.norm", "model.layers.0.input_layernorm",
                                   "model.layers.1.post_attention_layernorm", "model.layers.0.self_attn.q_norm", "model.layers.7.mlp"]])
def test_modules_that_stay_in_more_bits_anyway_may_be_named(key, names):
    """Embedding, head and norms are never 8-bit, and a layer that the model does not have keeps nothing."""
    from acvram_b200.config import Qwen3Config
    cfg = Qwen3Config.from_dict(fp8_config(**{key: names}))
    assert cfg.weights_fp8 and cfg == Qwen3Config.from_dict(fp8_config())


@pytest.mark.parametrize("names", ["q_proj", {"q_proj": True}, [3], ["re:.*q_proj"], ["model.layers.*"], [""]])
def test_a_list_that_cannot_be_read_is_refused(names):
    from acvram_b200.config import ConfigError, Qwen3Config
    with pytest.raises(ConfigError, match="a list of modules' names is read"):
        Qwen3Config.from_dict(fp8_config(modules_to_not_convert=names))


def test_the_list_of_another_method_is_not_read():
    from acvram_b200.config import Qwen3Config
    assert not Qwen3Config.from_dict(fp8_config(quant_method="other", modules_to_not_convert=["q_proj"])).weights_fp8


def test_weights_in_8_bits_are_not_asked_of_a_model_already_built():
    """Its weights would stay in more bits."""
    from acvram_b200 import Engine

    class Built:
        plan = None

        def forward(self):
            raise AssertionError

    with pytest.raises(ValueError, match="already built"):
        Engine(Built(), weights="fp8")


# ----------------------------------------------------------------------------- results whose rows overlap
def overlapping(t, by=1):
    """A view of t's memory with rows `by` elements less apart than they are long."""
    return t.as_strided(t.shape, (t.shape[1] - by, 1))


def test_results_whose_rows_overlap_are_refused():
    """Two rows' kernels would write the same elements, and the stream's be read by one when the other has written it."""
    import torch

    from acvram_b200.kernels import ops
    x, w = torch.zeros((4, 256)), torch.zeros(256)
    q, s = ops.fp8_rows(4, 256, "cpu")
    wq, ws = ops.fp8_rows(256, 256, "cpu")[0], torch.empty((2, 2))
    out = torch.empty((4, 256))
    one = lambda t: t[:1].expand(t.shape)
    calls = [(ops.quantize_fp8, (x, one(q), s), {}), (ops.quantize_fp8, (x, q, overlapping(s)), {}),
             (ops.quantize_fp8, (torch.zeros((256, 256)), wq, one(ws), 128), {}),
             (ops.linear_fp8, (q, s, wq, ws, one(out)), {}), (ops.linear_fp8, (q, s, wq, ws, overlapping(out)), {}),
             (ops.linear_fp8_swiglu, (q, s, wq, ws, wq, ws, overlapping(q), s), {}),
             (ops.linear_fp8_swiglu, (q, s, wq, ws, wq, ws, q, one(s)), {}),
             (ops.add_gated_norms, (one(x), x, q, s), {"weight": w}), (ops.add_gated_norms, (overlapping(x, 200), None, out), {"weight": w}),
             (ops.add_gated_norms, (x, x, overlapping(out), None), {"weight": w}), (ops.add_gated_norms, (x, x, one(q), s), {"weight": w}),
             (ops.add_gated_norms, (x, x, q, one(s)), {"weight": w})]
    for call, args, kw in calls:
        with pytest.raises(ops.KernelError, match="overlap"):
            call(*args, **kw)


def test_a_single_row_and_operands_that_are_only_read_may_have_any_stride():
    """These get as far as the question of the device."""
    import torch

    from acvram_b200.kernels import ops
    x, w = torch.zeros((4, 256)), torch.zeros(256)
    q, s = ops.fp8_rows(4, 256, "cpu")
    wq, ws = ops.fp8_rows(256, 256, "cpu")[0], torch.empty((2, 2))
    out = torch.empty((4, 256))
    one = lambda t: t[:1].expand(t.shape)
    narrow = lambda t: t.as_strided((1, t.shape[1]), (0, 1))
    calls = [(ops.quantize_fp8, (one(x), q, s), {}), (ops.quantize_fp8, (x[:1], narrow(q), narrow(s)), {}),
             (ops.linear_fp8, (q, one(s), wq, one(ws), out), {}), (ops.linear_fp8, (q[:1], s[:1], wq, ws, narrow(out)), {}),
             (ops.linear_fp8_swiglu, (q[:1], s[:1], wq, ws, wq, ws, narrow(q), narrow(s)), {}),
             (ops.add_gated_norms, (x, one(x), q, s), {"weight": w, "gate": one(x)}),
             (ops.add_gated_norms, (narrow(x), x[:1], narrow(q), narrow(s)), {"weight": w})]
    for call, args, kw in calls:
        with pytest.raises(ops.KernelError, match="CPU tensor"):
            call(*args, **kw)
