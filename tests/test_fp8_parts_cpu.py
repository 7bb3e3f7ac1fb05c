"""8-bit weights beside parts that know nothing of them."""

from __future__ import annotations

import pytest
import torch


def test_a_part_that_says_nothing_of_8_bit_rows_gets_the_norms_output():
    """Parts are registered by anyone, and need not be made from the package's base classes."""
    from acvram_b200.parts.blocks import PreNormBlock

    class Norm:
        groups = 1

        def forward(self, x, delta, **kw):
            return ("normed", kw)

        def forward_fp8(self, *args, **kw):
            raise AssertionError

    block = PreNormBlock.__new__(PreNormBlock)
    x = torch.zeros((2, 16))
    assert block._normed(Norm(), x, None, object(), {"out_dtype": torch.bfloat16}, {}) == ("normed", {"out_dtype": torch.bfloat16})


def attention(**kw):
    from acvram_b200.parts import PartSpec
    return PartSpec("attention", {"num_heads": 4, "num_kv_heads": 2, "head_dim": 16, "position": PartSpec("none", {}), "qk_norm_eps": None,
                                  "window": 0, **kw})


@pytest.mark.parametrize("mixer,ff", [({"fp8": True}, {}), ({}, {"fp8": True})])
def test_parts_whose_last_products_are_one_are_not_built_with_8_bit_weights(mixer, ff):
    from acvram_b200.parts import LayerSpec, PartSpec
    from acvram_b200.parts.registry import BLOCKS
    spec = LayerSpec("model.layers.0.", "parallel", attention(**mixer), PartSpec("swiglu", {"intermediate_size": 128, **ff}),
                                  PartSpec("rmsnorm", {"eps": 1e-6}))
    with pytest.raises(ValueError, match="8-bit weights cannot stand beside"):
        BLOCKS["parallel"](spec, 64)


def test_mixers_side_by_side_are_not_built_with_8_bit_weights():
    from acvram_b200.parts.registry import MIXERS
    for left, right in (({"fp8": True}, {}), ({}, {"fp8": True})):
        with pytest.raises(ValueError, match="8-bit weights cannot stand beside"):
            MIXERS["parallel"](64, attention(**left), attention(**right))
