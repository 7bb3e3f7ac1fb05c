"""The 8-bit operators of prompt sizes side by side: captured and replayed on two streams at once, and called on two streams at once."""

from __future__ import annotations

import pytest
import torch

from test_fp8_gpu import activations, chain, ops, quantized

pytestmark = pytest.mark.gpu
DEV = "cuda"


def run(x, wide):
    """Quantised weights, norm, gated product, product, and the rows of the stream quantised, in the form that their sizes ask for."""
    out = chain(x, wide, x.shape[0])
    q, s = ops().fp8_rows(*x.shape, DEV)
    ops().quantize_fp8(x, q, s)
    return out + [x, q.view(torch.uint8), s]


@pytest.mark.parametrize("T", [40, 600, 2300])
def test_whole_chains_on_two_streams(T):
    H, I = 512, 1280
    sides = [(activations(T, H, 4 + i, torch.bfloat16).to(DEV), (0.05 * activations(I, H, 3 + i)).to(DEV)) for i in range(2)]
    want = [[t.clone() for t in run(x.clone(), w)] for x, w in sides]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = []
        for i, (x, w) in enumerate(sides):
            with torch.cuda.stream(streams[i]):
                got.append(run(x.clone(), w))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    graphs, outs, xs = [], [], []
    for i, (x, w) in enumerate(sides):
        xs.append(x.clone())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(xs[i], w))
        graphs.append(g)
    for _ in range(10):
        for i in range(2):
            for t in outs[i]:
                t.zero_()
            xs[i].copy_(sides[i][0])            # (the norm changes the stream in place)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert ops().gemm_status() == 0


@pytest.mark.parametrize("gated", [False, True])
def test_pairs_of_ctas_on_two_streams(gated):
    """Both kernels want every multiprocessor and all of its tensor memory."""
    T, N, K = 2300, 3000, 640
    sides = []
    for i in range(2):
        x, xs = quantized(T, K, 1 + i, 1)
        w, ws = quantized(N, K, 3 + i, 128, 0.02)
        u, us = quantized(N, K, 5 + i, 128, 0.02)
        sides.append((x, xs, w, ws, u, us))

    def call(i):
        x, xs, w, ws, u, us = sides[i]
        if not gated:
            return [ops().linear_fp8(x, xs, w, ws, torch.empty((T, N), device=DEV), plan=(3, (256, 192)[i], 1))]
        q, s = ops().fp8_rows(T, N, DEV)
        ops().linear_fp8_swiglu(x, xs, w, ws, u, us, q, s, plan=(3, 256, 1))
        return [q.view(torch.uint8), s]

    want = [[t.clone() for t in call(i)] for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        got = [[], []]
        for i in (0, 1, 0, 1):
            with torch.cuda.stream(streams[i]):
                got[i] = call(i)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert ops().gemm_status() == 0
