"""The forms of the 8-bit operators that long prompts take, against their plain forms: norms of more rows than twice the multiprocessors,
quantised rows of more groups than the grid has half-warps (its loop, its steps of rows and groups, its double buffer, its last round)."""

from __future__ import annotations

import math

import pytest
import torch

import plain_fp8 as pf
from plain_fp8 import FP8, groups
from test_fp8_gpu import activations, check_norms, ops, same_bits

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("out_dtype", [F32, BF, FP8, None])
@pytest.mark.parametrize("stream,delta", [(F32, BF), (BF, BF), (F32, F32), (BF, F32)])
@pytest.mark.parametrize("T,H", [(297, 4096), (700, 1024), (300, 203)])
def test_norms_of_many_rows(T, H, stream, delta, out_dtype):
    check_norms(T, H, stream, delta, False, None, out_dtype)
    check_norms(T, H, stream, delta, True, "channels", out_dtype, 1)


@pytest.mark.parametrize("views", [False, True])
@pytest.mark.parametrize("gate", [None, "channels", F32, BF])
@pytest.mark.parametrize("post", [False, True])
def test_gated_norms_of_many_rows(post, gate, views):
    check_norms(300, 5120, F32, BF, post, gate, BF, 3, views)
    check_norms(298, 1032, BF, BF, post, gate, FP8, 4, views)
    check_norms(310, 1029, F32, F32, post, gate, FP8, 5, views)


@pytest.mark.parametrize("out_dtype", [BF, FP8])
@pytest.mark.parametrize("T,H", [(1000, 96), (2000, 127), (299, 8192), (299, 8200), (299, 8191), (297, 16384), (297, 16381), (5000, 1)])
def test_norms_of_many_rows_of_other_widths(T, H, out_dtype):
    check_norms(T, H, BF, BF, True, None, out_dtype, 6)
    check_norms(T, H, F32, None, False, None, out_dtype, 7)


def test_the_norm_in_front_of_a_prompts_products():
    """What the engine runs for every layer of a long prompt."""
    check_norms(2048, 4096, BF, BF, False, None, FP8, 8)
    check_norms(1023, 5120, F32, BF, False, None, FP8, 9)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("R,C", [(9473, 128), (9600, 200), (60_000, 100), (60_000, 72), (700, 8320), (900, 8320), (901, 8197), (1746, 5203), (7, 1_213_440),
                                 (5, 1_300_003)])
def test_quantize_of_many_groups_is_exact(R, C, dtype):
    x = activations(R, C, R + C, dtype)
    x[R // 2, C // 3] = float("nan")
    x[R - 1, C - 1] = float("inf")
    x[R - 2] = 0.0
    q, s = ops().fp8_rows(R, C, DEV)
    q.view(torch.uint8)[:] = 0x55
    s.fill_(3.0)
    ops().quantize_fp8(x.to(DEV), q, s)
    x = x.float()
    amax = torch.nn.functional.pad(x.abs(), (0, groups(C) * 128 - C)).view(R, -1, 128).amax(2)      # (a NaN is the largest of its group)
    want = pf.scale_of(amax)
    assert torch.equal(torch.nan_to_num(s.cpu(), nan=-1.0), torch.nan_to_num(want, nan=-1.0))
    codes = (x * (1.0 / want).repeat_interleave(128, 1)[:, :C]).clamp(-448.0, 448.0).to(FP8)
    assert same_bits(q, codes)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_behind_the_last_of_many_stay_as_they_were(dtype):
    R, C = 3000, 1000
    x = activations(R, C, 3, dtype).to(DEV)
    buf = torch.full((R + 3, 1040), 0x55, dtype=torch.uint8, device=DEV)
    sbuf = torch.full((R + 3, 9), 3.0, device=DEV)
    ops().quantize_fp8(x, buf.view(FP8)[:R, :C], sbuf[:R, :8])
    want = ops().quantize_fp8(x, *ops().fp8_rows(R, C, DEV))
    assert torch.equal(buf[:R, :C], want[0].view(torch.uint8)) and torch.equal(sbuf[:R, :8], want[1])
    assert bool((buf[R:] == 0x55).all()) and bool((buf[:, C:] == 0x55).all()) and bool((sbuf[R:] == 3.0).all()) and bool((sbuf[:, 8:] == 3.0).all())


# ----------------------------------------------------------------------------- the unit far from zero
@pytest.mark.parametrize("T,plan", [(3, (4, 16, 1)), (20, (4, 32, 1)), (3, (2, 256, 1)), (200, (2, 256, 1)), (300, (3, 256, 1))])
def test_gates_far_from_zero(T, plan):
    """Gates of -96 to 96, a group of units around each size, made without error (one term to a product, scales that are powers of two), so
    that what is off is the unit's own.  The exponential is off by 2 + 1.2 |g| units of a float (2 EPS32 each), which counts where g < 0; the
    quotient by two, one more each for the sum in the denominator, the product with the ups and the quotient's product with 1 / 448.  Beyond
    2^126 in the denominator (g under -87.3) the quotient is 0, where the value is under 1e-36."""
    centres = [-96.0, -88.0, -84.0, -60.0, -40.0, -20.0, -8.0, -2.0, 0.0, 2.0, 20.0, 96.0]
    I, K = 128 * len(centres), 128
    codes = torch.linspace(-240.0, 240.0, 481).to(FP8).float().unique()                     # numbers that e4m3 holds
    gates = torch.zeros((I, 1))
    scale = torch.ones((len(centres), 1))
    for i, c in enumerate(centres):
        scale[i] = 2.0 ** math.ceil(math.log2((abs(c) + 4.0) / 240.0))
        near = (codes * scale[i])[((codes * scale[i] - c).abs() <= max(4.0, abs(c) / 16))]
        gates[128 * i:128 * (i + 1), 0] = near[torch.arange(128) % len(near)] / scale[i]
    w = torch.zeros((I, K))
    w[:, :1] = gates
    u = torch.zeros((I, K))
    u[:, 1] = 1.0
    x = torch.zeros((T, K))
    x[:, :2] = 1.0

    def put(m):
        values, _ = ops().fp8_rows(*m.shape, DEV)
        values.view(torch.uint8).copy_(m.to(FP8).view(torch.uint8))
        return values

    out, s = ops().fp8_rows(T, I, DEV)
    ops().linear_fp8_swiglu(put(x), torch.ones((T, 1), device=DEV), put(w), scale.to(DEV), put(u), torch.ones((len(centres), 1), device=DEV),
                            out, s, plan=plan)
    g = (gates[:, 0] * scale.repeat_interleave(128, 0)[:, 0]).double().expand(T, I)
    h = g * torch.sigmoid(g)
    error = h.abs() * (2 + 1.2 * (-g).clamp(min=0) + 5) * 2 * pf.EPS32 + (g < -87.3) * h.abs()
    off = (pf.values(out, s, 1) - h).abs()
    bound = pf.quantized_error(h, s, error)
    assert bool((off <= bound).all()), float((off / bound).max())
    most = h.abs().view(T, -1, 128).amax(2) / 448
    most_error = error.view(T, -1, 128).amax(2) / 448
    assert bool(((s.cpu().double() - most).abs() <= most_error + most * 2 * pf.EPS32 + 2.0 ** -126).all())
