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
