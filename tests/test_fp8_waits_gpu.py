"""8-bit products whose bounded waits run out: whatever was asked for or issued by then has come to rest before the memory it uses goes
back, so the same kernel, run again at once, gives the right result.  K from one k-block to more than the stages hold: with few the loading
warp has asked for everything long before another warp gives up."""

from __future__ import annotations

import pytest
import torch

import plain_fp8 as pf

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ops():
    from acvram_b200.kernels import ops as module
    return module


def quantized(R, C, seed, block_rows):
    x = torch.randn((R, C), generator=torch.Generator().manual_seed(seed))
    q, s = pf.quantize(x, block_rows)
    values, _ = ops().fp8_rows(R, C, DEV)
    values.view(torch.uint8).copy_(q.view(torch.uint8))
    return values, s.to(DEV)


@pytest.mark.parametrize("k_blocks,skip", [(1, 0), (2, 1), (4, 0), (6, 5), (8, 0), (10, 9), (13, 6), (40, 39)])
@pytest.mark.parametrize("plan,gated,T,N", [((2, 128, 1), False, 200, 300), ((2, 128, 3), False, 200, 300), ((2, 256, 1), True, 200, 300),
                                            ((2, 256, 2), True, 200, 300), ((3, 256, 1), False, 300, 300), ((3, 192, 1), False, 300, 300),
                                            ((3, 256, 1), True, 300, 300), ((3, 256, 1), False, 2100, 2800), ((4, 16, 1), False, 16, 300),
                                            ((4, 16, 4), False, 16, 300), ((4, 32, 1), False, 32, 300), ((4, 32, 2), True, 32, 300)])
def test_nothing_is_under_way_when_a_product_gives_up(plan, gated, T, N, k_blocks, skip):
    K = 128 * k_blocks - 16
    x, xs = quantized(T, K, 1, 1)
    w, ws = quantized(N, K, 2, 128)

    def run():
        if gated:
            q, s = ops().fp8_rows(T, N, DEV)
            ops().linear_fp8_swiglu(x, xs, w, ws, w, ws, q, s, plan=plan)
            return q.view(torch.uint8).clone()
        return ops().linear_fp8(x, xs, w, ws, torch.empty((T, N), device=DEV), plan=plan)

    before = run()
    assert ops().gemm_status() == 0
    for _ in range(3):
        ops().gemm_fp8_test_fault(2000, skip)
        run()
        again = run()           # (behind it in the stream, with the full number of polls)
        assert ops().gemm_status() in (1, 2, 3, 4)
        ops().reset_after_failure()
        assert torch.equal(again, before) and ops().gemm_status() == 0
