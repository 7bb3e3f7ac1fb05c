"""The 8-bit operators against plain forms: quantisation bit for bit, products and norms within bounds that count roundings."""

from __future__ import annotations

import pytest
import torch

import plain_fp8 as pf
from plain_fp8 import EPS32, FP8, groups

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def ops():
    from acvram_b200.kernels import ops as module
    return module


def gen(seed):
    return torch.Generator().manual_seed(seed)


def activations(T, K, seed, dtype=F32):
    g = gen(seed)
    x = torch.randn((T, K), generator=g) * (0.3 + 2 * torch.rand((T, 1), generator=g))
    x[:, torch.randint(0, K, (1 + K // 200,), generator=g)] *= 20.0
    return x.to(dtype)


def device_pair(q, s, pad=0):
    """A quantised matrix on the device, rows at a stride of a multiple of 16 bytes and `pad` more."""
    R, C = q.shape
    buf = torch.full((R, (C + 15) // 16 * 16 + pad), 0x55, dtype=torch.uint8, device=DEV)
    buf[:, :C] = q.view(torch.uint8).to(DEV)
    return buf.view(FP8)[:, :C], s.to(DEV)


def quantized(R, C, seed, block_rows, factor=1.0, pad=0):
    q, s = pf.quantize(activations(R, C, seed) * factor, block_rows)
    return device_pair(q, s, pad)


def same_bits(a, b):
    a, b = a.cpu().view(torch.uint8), b.cpu().view(torch.uint8)
    nan = ((a & 0x7f) == 0x7f) & ((b & 0x7f) == 0x7f)
    return bool(((a == b) | nan).all())


# ----------------------------------------------------------------------------- quantisation
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("R,C", [(1, 1), (1, 128), (3, 7), (5, 130), (64, 96), (129, 264), (130, 1100), (257, 2048), (7, 12288), (2, 20001)])
def test_quantize_is_exact(R, C, block_rows, dtype):
    x = activations(R, C, R * 1000 + C, dtype)
    q, s = ops().fp8_rows(R, C, DEV)
    if block_rows == 128:
        s = torch.empty((groups(R), groups(C)), device=DEV)
    ops().quantize_fp8(x.to(DEV), q, s, block_rows)
    want_q, want_s = pf.quantize(x.float(), block_rows)
    assert torch.equal(s.cpu(), want_s)
    assert same_bits(q, want_q)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("offset,stride", [(0, 400), (1, 401), (8, 264), (16, 272)])
def test_quantize_views_leave_their_surroundings(block_rows, offset, stride):
    R, C = 37, 200
    base = torch.full((R + 2, stride), 7.0, dtype=BF, device=DEV)
    x = base[1:R + 1, offset:offset + C]
    x.copy_(activations(R, C, 5, BF))
    buf = torch.full((R + 2, stride + 3), 0x55, dtype=torch.uint8, device=DEV)
    q = buf.view(FP8)[1:R + 1, offset:offset + C]
    down = R if block_rows == 1 else 1
    sbuf = torch.full((down + 2, 5), 3.0, device=DEV)
    s = sbuf[1:down + 1, 1:3]
    ops().quantize_fp8(x, q, s, block_rows)
    want_q, want_s = pf.quantize(x.cpu().float(), block_rows)
    assert torch.equal(s.cpu(), want_s) and same_bits(q.contiguous(), want_q)
    buf.view(FP8)[1:R + 1, offset:offset + C].view(torch.uint8).fill_(0x55)
    s.fill_(3.0)
    assert bool((buf == 0x55).all()) and bool((sbuf == 3.0).all())


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantize_of_values_at_the_edges(block_rows, dtype):
    x = activations(6 if block_rows == 1 else 6 * 128, 384, 11)
    step = 1 if block_rows == 1 else 128
    x[0 * step:1 * step] = 0.0
    x[1 * step] = 1e-40                                     # under the smallest normal float
    x[2 * step, 130] = float("inf")
    x[3 * step, 5] = float("nan")
    x[4 * step] = torch.finfo(dtype).max
    x[5 * step, 200] = -float("inf")
    x = x.to(dtype)
    q, s = ops().fp8_rows(*x.shape, DEV)
    if block_rows == 128:
        s = torch.empty((groups(x.shape[0]), 3), device=DEV)
    ops().quantize_fp8(x.to(DEV), q, s, block_rows)
    want_q, want_s = pf.quantize(x.float(), block_rows)
    assert torch.equal(torch.nan_to_num(s.cpu(), nan=-1.0), torch.nan_to_num(want_s, nan=-1.0))
    assert same_bits(q, want_q)


# ----------------------------------------------------------------------------- the product
def check_product(T, N, K, out_dtype, seed, pads=(0, 0, 0), plan=None):
    x, xs = quantized(T, K, seed, 1, pad=16 * pads[0])
    w, ws = quantized(N, K, seed + 1, 128, 0.02, pad=16 * pads[1])
    buf = torch.full((T + 1, N + 1 + pads[2]), 7.0, dtype=out_dtype, device=DEV)
    out = buf[:T, :N]
    assert ops().linear_fp8(x, xs, w, ws, out, plan=plan) is out
    want, error = pf.product(x, xs, w, ws)
    if out_dtype != F32:
        error = error + pf.half_step(want.abs() + error, out_dtype)
    else:
        error = error + pf.half_step(want, F32)
    off = (out.cpu().double() - want).abs()
    assert bool((off <= error).all()), float((off / error).max())
    assert bool((buf[T:] == 7.0).all()) and bool((buf[:, N:] == 7.0).all())


@pytest.mark.parametrize("out_dtype", [BF, F32])
@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 16, 17, 33, 64, 65, 100, 128, 129, 200, 257, 300, 520])
@pytest.mark.parametrize("N,K", [(128, 128), (136, 144), (1000, 1104), (257, 2048)])
def test_product(T, N, K, out_dtype):
    check_product(T, N, K, out_dtype, T * 7 + N)


@pytest.mark.parametrize("T,N,K", [(1, 1, 16), (1, 5, 1), (3, 16, 100), (9, 31, 48), (1, 4096, 4096), (8, 640, 12288), (16, 1024, 5120),
                                   (40, 7, 4096), (130, 1, 256), (70, 130, 17408), (600, 2049, 272), (1024, 520, 640), (2050, 384, 512)])
def test_product_of_other_sizes(T, N, K):
    check_product(T, N, K, F32, T + N + K, (1, 2, 3))


@pytest.mark.parametrize("plan", [(1, 0, 1), (2, 128, 1), (2, 128, 2), (2, 128, 8), (3, 256, 1), (3, 224, 1), (3, 192, 1), (4, 16, 1), (4, 16, 8), (4, 32, 2)])
@pytest.mark.parametrize("T,N,K,out_dtype", [(16, 257, 2048, F32), (1, 128, 128, F32), (5, 300, 400, BF), (140, 130, 1100, F32), (300, 700, 2048, BF), (513, 257, 1296, F32)])
def test_product_by_every_plan(T, N, K, out_dtype, plan):
    if plan[0] == 1 and T > 16:
        with pytest.raises(ops().KernelError, match="outside what this kernel takes"):
            check_product(T, N, K, out_dtype, T + 3, plan=plan)
        return
    check_product(T, N, K, out_dtype, T + 3, plan=plan)


def test_products_of_many_tiles():
    """More tiles than multiprocessors, so that a pair of CTAs walks several."""
    for columns in (256, 224, 192):
        check_product(1500, 6000, 272, BF, 5, plan=(3, columns, 1))
    check_gated(1500, 4000, 272, 5, plan=(3, 256, 1))


@pytest.mark.parametrize("T", [1, 12, 90, 400])
def test_product_of_values_that_are_no_numbers(T):
    """A NaN or an infinity in a token's group, or an infinite scale, reaches that token's outputs and no other's."""
    N, K = 200, 400
    a = activations(T, K, 3)
    if T > 2:
        a[1, 300] = float("inf")
        a[T - 1, 2] = float("nan")
    x, xs = device_pair(*pf.quantize(a, 1))
    w, ws = quantized(N, K, 4, 128, 0.02)
    out = torch.empty((T, N), device=DEV)
    ops().linear_fp8(x, xs, w, ws, out)
    bad = torch.isnan(out).all(1).cpu()
    some = torch.isnan(out).any(1).cpu()
    want = torch.zeros(T, dtype=torch.bool)
    if T > 2:
        want[1] = want[T - 1] = True
    assert torch.equal(bad, want) and torch.equal(some, want)


# ----------------------------------------------------------------------------- the product with the gated unit
def check_gated(T, I, K, seed, gate_factor=0.05, plan=None):
    x, xs = quantized(T, K, seed, 1)
    g, gs = quantized(I, K, seed + 1, 128, gate_factor)
    u, us = quantized(I, K, seed + 2, 128, 0.02)
    buf = torch.full((T + 1, (I + 15) // 16 * 16 + 16), 0x55, dtype=torch.uint8, device=DEV)
    out = buf.view(FP8)[:T, :I]
    sbuf = torch.full((T + 1, groups(I) + 1), 3.0, device=DEV)
    scales = sbuf[:T, :groups(I)]
    ops().linear_fp8_swiglu(x, xs, g, gs, u, us, out, scales, plan=plan)
    yg, eg = pf.product(x, xs, g, gs)
    yu, eu = pf.product(x, xs, u, us)
    h = yg * torch.sigmoid(yg) * yu
    # the unit's slope is at most 1.1; the exponential, the quotient and the product are a few units of a float
    error = 1.1 * eg * (yu.abs() + eu) + (yg * torch.sigmoid(yg)).abs() * eu + h.abs() * 16 * EPS32
    off = (pf.values(out, scales, 1) - h).abs()
    bound = pf.quantized_error(h, scales, error)
    assert bool((off <= bound).all()), float((off / bound).max())
    pad = groups(I) * 128 - I
    most = torch.nn.functional.pad(h.abs(), (0, pad)).view(T, -1, 128).amax(2) / 448
    most_error = torch.nn.functional.pad(error, (0, pad)).view(T, -1, 128).amax(2) / 448
    assert bool(((scales.cpu().double() - most).abs() <= most_error + most * 2 * EPS32 + 2.0 ** -126).all())
    assert bool((buf[T:] == 0x55).all()) and bool((buf[:, I:] == 0x55).all())
    assert bool((sbuf[T:] == 3.0).all()) and bool((sbuf[:, groups(I):] == 3.0).all())


@pytest.mark.parametrize("T", [1, 5, 8, 9, 16, 17, 40, 64, 65, 128, 129, 300])
@pytest.mark.parametrize("I,K", [(128, 128), (200, 144), (1, 16), (1030, 1104), (640, 2048)])
def test_gated_product(T, I, K):
    check_gated(T, I, K, T + I)


@pytest.mark.parametrize("T,I,K", [(1, 4096, 4096), (4, 300, 12288), (70, 130, 5120), (520, 2049, 272), (1030, 384, 640)])
def test_gated_product_of_other_sizes(T, I, K):
    check_gated(T, I, K, T + I + K)


@pytest.mark.parametrize("plan", [(2, 256, 1), (2, 256, 2), (2, 256, 5), (3, 256, 1), (4, 16, 1), (4, 16, 3), (4, 32, 2), (4, 32, 4)])
@pytest.mark.parametrize("T,I,K", [(1, 128, 128), (5, 300, 400), (140, 130, 1100), (300, 700, 2048), (513, 257, 1296)])
def test_gated_product_by_every_plan(T, I, K, plan):
    check_gated(T, I, K, T + 3, plan=plan)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("kind", [2, 3, 4])
def test_a_wait_that_runs_out_is_reported(kind, gated):
    """A product whose producer leaves out a k-block gives up after a few polls, says so in the status word, and the next one runs."""
    x, xs = quantized(200, 1024, 1, 1)
    w, ws = quantized(300, 1024, 2, 128)
    plan = (kind, 32 if kind == 4 else 256 if gated or kind == 3 else 128, 1)

    def run():
        if gated:
            q, s = ops().fp8_rows(200, 300, DEV)
            ops().linear_fp8_swiglu(x, xs, w, ws, w, ws, q, s, plan=plan)
            return q.float()
        return ops().linear_fp8(x, xs, w, ws, torch.empty((200, 300), device=DEV), plan=plan)

    before = run()
    assert ops().gemm_status() == 0
    ops().gemm_fp8_test_fault(2000, 3)
    run()
    torch.cuda.synchronize()
    assert ops().gemm_status() in (1, 2, 3, 4)
    ops().reset_after_failure()
    assert ops().gemm_status() == 0
    assert torch.equal(run(), before) and ops().gemm_status() == 0


# ----------------------------------------------------------------------------- the norms
def check_norms(T, H, stream, delta, post, gate, out_dtype, seed=0, views=False):
    g = gen(seed + T * 31 + H)
    def matrix(values, dtype, extra):
        if not views:
            return values.to(dtype).to(DEV)
        buf = torch.full((T, H + extra), 9.0, dtype=dtype, device=DEV)
        buf[:, :H] = values.to(dtype)
        return buf[:, :H]
    x = matrix(3 * activations(T, H, seed + 1), stream, 24)
    d = matrix(0.5 * activations(T, H, seed + 2), delta, 8) if delta is not None else None
    w1 = (1 + 0.2 * torch.randn(H, generator=g)).to(DEV) if post else None
    w2 = (1 + 0.2 * torch.randn(H, generator=g)).to(DEV)
    gv = None
    if gate == "channels":
        gv = torch.randn(H, generator=g).to(DEV)
    elif gate is not None:
        gv = matrix(torch.randn((T, H), generator=g), gate, 16)
    c = 0.7
    x0 = x.cpu().double()
    if out_dtype == FP8:
        out, scales = ops().fp8_rows(T, H, DEV)
    else:
        out, scales = (torch.empty((T, H), dtype=out_dtype, device=DEV) if out_dtype is not None else None), None
    ops().add_gated_norms(x, d, out, scales, post_weight=w1, post_eps=1e-5, gate=gv, residual_scale=c,
                          weight=w2 if out is not None else None, eps=1e-6)
    # a sum of H squares by a thread's sixteen to 64 and then by ten halvings: at most 80 roundings, half of which the root keeps;
    # the products in front of and behind it are six more
    rounds = 50 * EPS32
    want = x0
    error = torch.zeros_like(x0)
    if d is not None:
        n = d.cpu().double()
        if w1 is not None:
            n = n / torch.sqrt(n.square().mean(1, keepdim=True) + 1e-5) * w1.cpu().double()
        if gv is not None:
            n = n * gv.cpu().double()
        want = x0 + c * n
        error = (c * n).abs() * rounds + (want.abs() + (c * n).abs() * rounds) * EPS32
        if stream != F32:
            error = error + pf.half_step(want.abs() + error, stream)
    kept = x.cpu().double()
    assert bool(((kept - want).abs() <= error).all())
    if out is None:
        return
    h = kept / torch.sqrt(kept.square().mean(1, keepdim=True) + 1e-6) * w2.cpu().double()
    error = h.abs() * rounds
    if out_dtype == FP8:
        off, bound = (pf.values(out, scales, 1) - h).abs(), pf.quantized_error(h, scales, error)
        most = torch.nn.functional.pad(h.abs(), (0, groups(H) * 128 - H)).view(T, -1, 128).amax(2) / 448
        assert bool(((scales.cpu().double() - most).abs() <= most * (rounds + 2 * EPS32) + 2.0 ** -126).all())
    else:
        off, bound = (out.cpu().double() - h).abs(), error + pf.half_step(h.abs() + error, out_dtype)
    assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("out_dtype", [F32, BF, FP8, None])
@pytest.mark.parametrize("stream", [F32, BF])
@pytest.mark.parametrize("T,H", [(1, 1), (3, 96), (2, 127), (5, 1024), (8, 4096), (3, 5120), (2, 8200), (2, 16384)])
def test_norms(T, H, stream, out_dtype):
    check_norms(T, H, stream, BF, True, None, out_dtype)


@pytest.mark.parametrize("views", [False, True])
@pytest.mark.parametrize("gate", [None, "channels", F32, BF])
@pytest.mark.parametrize("delta,post", [(F32, False), (F32, True), (BF, False), (BF, True)])
def test_norms_with_gates(delta, post, gate, views):
    check_norms(6, 1032, F32, delta, post, gate, FP8, 3, views)
    check_norms(4, 203, BF, delta, post, gate, BF, 4, views)


@pytest.mark.parametrize("out_dtype", [F32, BF, FP8])
def test_norm_without_a_part(out_dtype):
    check_norms(5, 640, BF, None, False, None, out_dtype)
    check_norms(5, 6000, F32, None, False, None, out_dtype)


def test_norms_of_rows_of_zeros():
    H = 256
    x, d = torch.zeros((2, H), device=DEV), torch.zeros((2, H), device=DEV)
    w = torch.ones(H, device=DEV)
    q, s = ops().fp8_rows(2, H, DEV)
    ops().add_gated_norms(x, d, q, s, post_weight=w, post_eps=1e-6, weight=w, eps=1e-6)
    assert bool((x == 0).all()) and bool((q.float() == 0).all()) and bool((s == 2.0 ** -126).all())


# ----------------------------------------------------------------------------- calls one behind the other
def chain(x, wide, T):
    """Quantised weights, norm, gated product, product, as a step runs them, everything made by the kernel in front."""
    o = ops()
    H, I = x.shape[1], wide.shape[0]
    g, gs = o.fp8_rows(I, H, DEV)[0], torch.empty((groups(I), groups(H)), device=DEV)
    o.quantize_fp8(wide, g, gs, 128)
    q, s = o.fp8_rows(T, H, DEV)
    o.add_gated_norms(x, x.clone(), q, s, weight=torch.ones(H, device=DEV), eps=1e-6)
    a, b = o.fp8_rows(T, I, DEV)
    o.linear_fp8_swiglu(q, s, g, gs, g, gs, a, b)
    d, ds = o.fp8_rows(H, I, DEV)[0], torch.empty((groups(H), groups(I)), device=DEV)
    o.quantize_fp8(wide.t().contiguous(), d, ds, 128)
    out = torch.empty((T, H), device=DEV)
    o.linear_fp8(a, b, d, ds, out)
    return [t.clone() for t in (q.view(torch.uint8), s, a.view(torch.uint8), b, out)]


@pytest.mark.parametrize("T", [1, 16, 30, 100, 600])
def test_a_chain_whose_every_input_is_made_by_the_kernel_in_front(T):
    """Kernels begin while the one in front still runs: run without a pause the chain gives what it gives with a wait behind every call."""
    H, I = 512, 1280
    wide = (0.05 * activations(I, H, 3)).to(DEV)
    x0 = activations(T, H, 4, BF).to(DEV)
    import contextlib

    @contextlib.contextmanager
    def waiting():
        o = ops()
        real = o._launch_record
        def launch(*args):
            real(*args)
            torch.cuda.synchronize()
        o._launch_record = launch
        try:
            yield
        finally:
            o._launch_record = real

    with waiting():
        want = chain(x0.clone(), wide, T)
    for _ in range(20):
        for a, b in zip(chain(x0.clone(), wide, T), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [1, 12, 40, 300])
def test_captured_and_on_two_streams(T):
    """Two captured graphs and two streams at once share nothing but the status word."""
    K, N = 1024, 640
    x, xs = quantized(T, K, 1, 1)
    sets = []
    for i in range(2):
        w, ws = quantized(N, K, 2 + i, 128, 0.02)
        u, us = quantized(N, K, 8 + i, 128, 0.02)
        sets.append((w, ws, u, us))

    def run(i):
        w, ws, u, us = sets[i]
        out = torch.empty((T, N), device=DEV)
        ops().linear_fp8(x, xs, w, ws, out, static_weights=True)
        q, s = ops().fp8_rows(T, N, DEV)
        ops().linear_fp8_swiglu(x, xs, w, ws, u, us, q, s, static_weights=True)
        return out, q.view(torch.uint8), s

    want = [[t.clone() for t in run(i)] for i in range(2)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(i))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for i in (0, 1):
            for t in outs[i]:
                t.zero_() if t.dtype != torch.uint8 else t.fill_(0)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            for a, b in zip(outs[i], want[i]):
                assert torch.equal(a, b)
    for _ in range(10):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(run(i))
        torch.cuda.synchronize()
        for i in (0, 1):
            for a, b in zip(got[i], want[i]):
                assert torch.equal(a, b)
    assert ops().gemm_status() == 0


# ----------------------------------------------------------------------------- the ends of the range
def test_rows_that_are_not_on_16_bytes_are_refused():
    x, xs = quantized(4, 256, 1, 1)
    w, ws = quantized(8, 256, 2, 128)
    out = torch.empty((4, 8), device=DEV)
    flat = torch.zeros(4 * 264 + 1, dtype=torch.uint8, device=DEV).view(FP8)
    for bad in (flat[:4 * 264].view(4, 264)[:, :256], flat[1:1 + 4 * 256].view(4, 256), x[:1].expand(4, 256), flat.as_strided((4, 256), (16, 1))):
        with pytest.raises(ops().KernelError, match="aligned"):
            ops().linear_fp8(bad, xs, w, ws, out)
    bad = torch.zeros((8, 264), dtype=torch.uint8, device=DEV).view(FP8)[:, :256]
    with pytest.raises(ops().KernelError, match="aligned"):
        ops().linear_fp8(x, xs, bad, ws, out)
    q, s = ops().fp8_rows(4, 8, DEV)
    for g, u in ((w, bad), (bad, w)):
        with pytest.raises(ops().KernelError, match="aligned"):
            ops().linear_fp8_swiglu(x, xs, g, ws, u, ws, q, s)


@pytest.mark.parametrize("plan", [None, (2, 128, 1), (4, 16, 1)])
def test_a_single_row_has_no_stride(plan):
    x, xs = quantized(3, 250, 1, 1)
    w, ws = quantized(1, 250, 2, 128)
    want = ops().linear_fp8(x[:1], xs[:1], w, ws, torch.empty((1, 1), device=DEV), plan=plan)
    got = ops().linear_fp8(x[:1].clone(memory_format=torch.contiguous_format), xs[:1], w.as_strided((1, 250), (3, 1)), ws,
                           torch.empty((1, 1), device=DEV), plan=plan)
    assert torch.equal(want, got)


def test_no_tokens_no_features_and_no_inner_elements():
    e = lambda r, c, dt=F32: torch.empty((r, c), device=DEV, dtype=dt)
    w, ws = quantized(8, 256, 2, 128)
    assert ops().linear_fp8(e(0, 256, FP8), e(0, 2), w, ws, e(0, 8)).shape == (0, 8)
    x, xs = quantized(4, 256, 1, 1)
    assert ops().linear_fp8(x, xs, e(0, 256, FP8), e(0, 2), e(4, 0)).shape == (4, 0)
    out = torch.full((4, 8), 5.0, device=DEV)
    ops().linear_fp8(e(4, 0, FP8), e(4, 0), e(8, 0, FP8), e(1, 0), out)
    assert bool((out == 0).all())
    with pytest.raises(ops().KernelError, match="K is 0"):
        ops().linear_fp8_swiglu(e(4, 0, FP8), e(4, 0), e(8, 0, FP8), e(1, 0), e(8, 0, FP8), e(1, 0), e(4, 8, FP8), e(4, 1))
    ops().quantize_fp8(e(0, 256), e(0, 256, FP8), e(0, 2))
    ops().add_gated_norms(e(0, 256), None, e(0, 256), weight=torch.ones(256, device=DEV))
    torch.cuda.synchronize()


def test_a_row_wider_than_a_block_holds_is_refused():
    H = ops().GATED_NORMS_WIDTH + 8
    x = torch.ones((2, H), device=DEV)
    with pytest.raises(ops().KernelError, match="outside what this kernel takes"):
        ops().add_gated_norms(x, None, torch.empty_like(x), weight=torch.ones(H, device=DEV))


@pytest.mark.parametrize("T,K", [(1, 100_000), (20, 70_000), (32, 400_000)])
def test_products_of_long_rows(T, K):
    """Rows whose scales would not fit a tile's shared memory take a plan that holds none."""
    check_product(T, 130, K, F32, T)
    check_gated(T, 130, K, T, gate_factor=0.005)


def test_matrices_of_more_than_2_to_the_31():
    """More than 2^31 elements in a matrix: its last rows are right."""
    T, N, K = 65_700, 32_800, 128
    x, xs = quantized(300, K, 1, 1)
    big_x, big_xs = ops().fp8_rows(T, K, DEV)
    big_x.view(torch.uint8)[:] = 0
    big_xs.fill_(1.0)
    big_x.view(torch.uint8)[-300:] = x.view(torch.uint8)
    big_xs[-300:] = xs
    w, ws = quantized(N, K, 2, 128, 0.02)
    out = torch.empty((T, N), device=DEV, dtype=BF)
    ops().linear_fp8(big_x, big_xs, w, ws, out)
    want, error = pf.product(x, xs, w, ws)
    alone = out[-300:].clone()
    assert bool(((alone.cpu().double() - want).abs() <= error + pf.half_step(want.abs() + error, BF)).all())
    assert not bool(out[:1000].any())
    q, s = ops().fp8_rows(T, N, DEV)
    ops().quantize_fp8(out, q, s)
    q1, s1 = ops().fp8_rows(300, N, DEV)
    ops().quantize_fp8(alone, q1, s1)
    assert torch.equal(q[-300:].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[-300:], s1)
    blocks = torch.empty((groups(T), groups(N)), device=DEV)
    ops().quantize_fp8(out, q, blocks, 128)
    tail = T // 128 * 128
    q1, s1 = ops().fp8_rows(T - tail, N, DEV)
    last = torch.empty((1, groups(N)), device=DEV)
    ops().quantize_fp8(out[tail:], q1, last, 128)
    assert torch.equal(q[tail:].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(blocks[-1:], last)
    del out, q, q1
    rows = 140_000
    stream = torch.zeros((rows, 16384), device=DEV, dtype=BF)
    stream[-3:] = activations(3, 16384, 3, BF).to(DEV)
    weight = torch.ones(16384, device=DEV)
    q, s = ops().fp8_rows(rows, 16384, DEV)
    ops().add_gated_norms(stream, None, q, s, weight=weight, eps=1e-6)
    want = stream[-3:].double()
    want = (want / torch.sqrt(want.square().mean(1, keepdim=True) + 1e-6)).cpu()
    off = (pf.values(q[-3:], s[-3:], 1) - want).abs()
    assert bool((off <= pf.quantized_error(want, s[-3:], want.abs() * 50 * EPS32)).all())
    assert not bool(q[:3].view(torch.uint8).any())
