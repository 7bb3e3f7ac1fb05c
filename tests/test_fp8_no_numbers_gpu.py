"""Rows that hold a NaN or an infinity, through every form of the gated product and of the norms: they reach no other row, and what they
leave is what the definition says."""

from __future__ import annotations

import pytest
import torch

import plain_fp8 as pf
from plain_fp8 import FP8, groups
from test_fp8_gpu import activations, device_pair, ops, quantized

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("I", [128, 200, 640])
@pytest.mark.parametrize("T,plan", [(5, None), (12, (4, 16, 1)), (12, (4, 16, 3)), (30, (4, 32, 2)), (90, (2, 256, 1)), (90, (2, 256, 3)),
                                    (400, (3, 256, 1)), (1000, None)])
def test_gated_product_of_values_that_are_no_numbers(T, plan, I):
    K = 400
    a = activations(T, K, 3)
    a[1, 300] = float("inf")
    a[T - 1, 2] = float("nan")
    x, xs = device_pair(*pf.quantize(a, 1))
    g, gs = quantized(I, K, 4, 128, 0.02)
    u, us = quantized(I, K, 5, 128, 0.02)
    out, s = ops().fp8_rows(T, I, DEV)
    ops().linear_fp8_swiglu(x, xs, g, gs, u, us, out, s, plan=plan)
    good = torch.ones(T, dtype=torch.bool)
    good[1] = good[T - 1] = False
    v, s = out.cpu().float(), s.cpu()
    assert bool(torch.isnan(v[~good]).all()) and bool(torch.isnan(s[~good]).all())
    assert bool(torch.isfinite(v[good]).all()) and bool(torch.isfinite(s[good]).all())
    # the others are what they are without them, bit for bit
    clean = activations(T, K, 3)
    clean[~good] = 0.0
    x, xs = device_pair(*pf.quantize(clean, 1))
    out0, s0 = ops().fp8_rows(T, I, DEV)
    ops().linear_fp8_swiglu(x, xs, g, gs, u, us, out0, s0, plan=plan)
    assert torch.equal(out0.cpu().view(torch.uint8)[good], out.cpu().view(torch.uint8)[good]) and torch.equal(s0.cpu()[good], s[good])


@pytest.mark.parametrize("out_dtype", [F32, BF, FP8])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("T,H", [(6, 640), (6, 203), (4, 8200), (300, 1024), (300, 1029)])
def test_norms_of_values_that_are_no_numbers(T, H, post, out_dtype):
    """A NaN in the part or the stream makes the row's result NaN; an infinity in the stream zeroes the row's finite elements and is NaN itself
    (it is divided by its own size), and so, quantised, its group; in the part, behind which a norm stands, the same happens to what joins the
    stream.  The stream keeps what the sum gives."""
    x0, d0 = activations(T, H, 1), activations(T, H, 2)
    x0[0, 5], d0[1, 7], x0[2, 150], d0[3, 150] = float("nan"), float("nan"), float("inf"), float("inf")
    x, d = x0.to(DEV), d0.to(DEV)
    w = torch.ones(H, device=DEV)
    if out_dtype == FP8:
        out, s = ops().fp8_rows(T, H, DEV)
    else:
        out, s = torch.empty((T, H), device=DEV, dtype=out_dtype), None
    ops().add_gated_norms(x, d, out, s, post_weight=w if post else None, post_eps=1e-6, weight=w, eps=1e-6)
    n = d0.double()
    if post:
        n = n / torch.sqrt(n.square().mean(1, keepdim=True) + 1e-6)
    kept = x0.double() + n
    stream = x.cpu()
    assert torch.equal(torch.isnan(stream), torch.isnan(kept)) and torch.equal(torch.isinf(stream), torch.isinf(kept))
    h = kept / torch.sqrt(kept.square().mean(1, keepdim=True) + 1e-6)
    if out_dtype != FP8:
        assert torch.equal(torch.isnan(out.cpu()), torch.isnan(h)) and not bool(torch.isinf(out.cpu()).any())
        return
    bad = torch.isnan(torch.nn.functional.pad(h, (0, groups(H) * 128 - H))).view(T, -1, 128).any(2)     # a NaN takes its group with it
    assert torch.equal(torch.isnan(s.cpu()), bad)
    assert torch.equal(torch.isnan(out.cpu().float()), bad.repeat_interleave(128, 1)[:, :H])
