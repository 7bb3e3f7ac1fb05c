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
