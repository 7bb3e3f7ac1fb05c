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
    assert ops._NORMS_ARGS.size == 9 * 8 + 5 * 8 + 7 * 4 + 3 * 4


def test_plain_quantisation_is_near_what_it_stands_for():
    x = torch.randn((200, 300), generator=torch.Generator().manual_seed(1))
    for block_rows in (1, 128):
        q, s = pf.quantize(x, block_rows)
        off = (pf.values(q, s, block_rows) - x.double()).abs()
        assert bool((off <= x.double().abs() * 2.0 ** -4 * (1 + 1e-6) + pf.spread(s.double(), 200, 300, block_rows) * 2.0 ** -10).all())
