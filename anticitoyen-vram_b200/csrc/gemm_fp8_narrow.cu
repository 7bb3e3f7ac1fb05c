// The products of e4m3 operands with block scales for few tokens on the fifth-generation tensor cores: weight rows are the tensor core's
// rows (128 to a tile, so a tile is one block row of their scales), tokens its columns.
//
// The mathematics are those of gemm_fp8_tc.cu: a k-block's products come to rest in tensor memory, and the epilogue adds them, times
// their scales, to the float sums in its registers.  What bounds it is the stream of weights: nothing but them and the few tokens
// passes through shared memory, and K is split over the CTAs of a cluster so that as many tiles are under way as fit the SMs at once.
// A lane holds a weight row, so a column's scale sx[t][g] sw[g] is the same for all: the products of the two are made once, into shared
// memory, and read four at a time.  In the gated form a tile is 64 units' gate rows and their up rows, a cluster has a tile for either
// half of a group of 128 units, and meets to write it.
#include "fp8_tc.cuh"

#define FN_THREADS 192                      // two warps to load and to issue, four of epilogue
template <int BT>
struct Fp8NarrowShape {
    static constexpr int STAGE = FT_TILE + BT * FT_ROWS;
    static constexpr int RESIDENT = 3;                                      // CTAs to an SM at most
    static constexpr int SLOTS = 4;                                         // partial results in tensor memory
    static constexpr int TMEM = SLOTS * BT;
    // registers of a thread: they are handed out for warps rounded up to four
    static constexpr int REGS = 65536 / RESIDENT / 256 / 8 * 8;
    static constexpr int LD = FT_ROWS + 4;                                  // floats between two tokens' sums
    static constexpr int SUMS = (BT * LD * 4 + 1023) / 1024 * 1024;
};

template <int BT, bool GATED>
__global__ void __launch_bounds__(FN_THREADS) __maxnreg__(Fp8NarrowShape<BT>::REGS)
gemm_fp8_narrow_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                       const __grid_constant__ CUtensorMap map_w2, const Fp8TcParams p) {
    using S = Fp8NarrowShape<BT>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* tiles = smem_raw + ((1024u - (gt_smem(smem_raw) & 1023u)) & 1023u);
    const int STAGES = p.stages;
    const uint32_t tiles_addr = gt_smem(tiles);
    const int area = STAGES * S::STAGE > S::SUMS ? STAGES * S::STAGE : S::SUMS;
    const uint32_t full0 = tiles_addr + area, empty0 = full0 + 8 * STAGES, tfull0 = empty0 + 8 * STAGES, tempty0 = tfull0 + 8 * S::SLOTS;
    float* scales = reinterpret_cast<float*>(tiles + area + 256);           // [k-block][64 rows each of gate and up, or one for all][token]
    __shared__ uint32_t tmem_base_s;
    __shared__ volatile int abort_s;
    __shared__ int asked_s, issued_s;           // k-blocks whose loads and whose products are issued
    const int warp = ft_warp(), lane = threadIdx.x & 31;
    constexpr int HALVES = GATED ? 2 : 1;
    const int size = p.splits * HALVES, rank = blockIdx.x % size, split = rank / HALVES, half = rank % HALVES;
    const int tile = blockIdx.x / size, ta = tile % p.tiles_m, tb = tile / p.tiles_m;
    const int kb0 = split * p.kb_per_split, kb1 = min(kb0 + p.kb_per_split, p.n_kb), t0 = ta * BT;
    // Each tile begins at another of its k-blocks and goes round: the CTAs, which start together, would all read the same tokens' bytes
    // at the same time (a tile's order is its own, whatever the others do).
    const int count = kb1 - kb0, turned = (int)(ft_spread(tb * HALVES + half) % (unsigned)count);
    auto block_of = [&](int i) { return i + turned < count ? i + turned : i + turned - count; };
    if (threadIdx.x == 0) {
        abort_s = 0;
        for (int s = 0; s < STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int b = 0; b < S::SLOTS; ++b) { mbar_init(tfull0 + 8 * b, 1); mbar_init(tempty0 + 8 * b, 4); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(gt_smem(&tmem_base_s)), "r"(S::TMEM));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_s;
    // (only now may the next kernel's CTAs come: one that took tensor memory before this CTA had its own could wait for this grid)
    pdl_launch_dependents();

    bool failed = false;            // this warp gave up a wait
    if (warp == 0) {
        auto load_w = [&](int s, int kb) {
            tma_load_2d(tiles_addr + s * S::STAGE, &map_w, full0 + 8 * s, kb * FT_ROWS, tb * FT_ROWS + half * 64);
            if (GATED) tma_load_2d(tiles_addr + s * S::STAGE + FT_TILE / 2, &map_w2, full0 + 8 * s, kb * FT_ROWS, tb * FT_ROWS + half * 64);
        };
        const int early = p.early_w ? min(STAGES, count) : 0;
        if (ft_elect()) {
            for (int i = 0; i < early; ++i) {
                mbar_expect_tx(full0 + 8 * i, S::STAGE);
                load_w(i, kb0 + block_of(i));
            }
        }
        __syncwarp();
        pdl_wait();
        int s = 0, asked = 0;
        uint32_t ph = 0;
        bool ready = false;
        for (; asked < count; ++asked) {
            const bool half_done = asked < early;
            const int kb = kb0 + block_of(asked);
            if (!half_done && !ready) {
                failed = ft_warp_failed(empty0 + 8 * s, ph ^ 1, &abort_s, p, 1);
                if (failed) break;
            }
            if (ft_elect()) {
                if (!half_done) mbar_expect_tx(full0 + 8 * s, S::STAGE);
                if (kb != p.skip_kb) {
                    tma_load_2d(tiles_addr + s * S::STAGE + FT_TILE, &map_x, full0 + 8 * s, kb * FT_ROWS, t0);
                    if (!half_done) load_w(s, kb);
                }
            }
            __syncwarp();
            if (++s == STAGES) { s = 0; ph ^= 1; }
            ready = __all_sync(0xffffffffu, ft_ready(empty0 + 8 * s, ph ^ 1));
        }
        if (lane == 0) asked_s = asked;
    } else if (warp == 1) {
        pdl_wait();
        const uint32_t idesc = ft_idesc(BT, FT_ROWS);
        const uint64_t a0 = umma_desc(tiles_addr), b0 = umma_desc(tiles_addr + FT_TILE);
        uint32_t ph = 0;
        int s = 0;
        bool ready = false;
        int i = 0;
        for (; i < count; ++i) {
            const uint32_t slot = (uint32_t)i % S::SLOTS, use = (uint32_t)i / S::SLOTS;
            if ((!ready && ft_warp_failed(full0 + 8 * s, ph, &abort_s, p, 3)) ||
                (use && ft_warp_failed(tempty0 + 8 * slot, (use & 1) ^ 1, &abort_s, p, 2)))
                break;
            tc_fence_after();
            if (ft_elect()) {
                const uint64_t a = a0 + (uint64_t)(s * (S::STAGE >> 4)), b = b0 + (uint64_t)(s * (S::STAGE >> 4));
#pragma unroll
                for (int k = 0; k < 4; ++k) ft_mma<false>(tmem_base + slot * BT, a + 2 * k, b + 2 * k, idesc, k > 0);
                tc_commit(tfull0 + 8 * slot);
                tc_commit(empty0 + 8 * s);
            }
            __syncwarp();
            if (++s == STAGES) { s = 0; ph ^= 1; }
            ready = __all_sync(0xffffffffu, ft_ready(full0 + 8 * s, ph));
        }
        failed = i < count;
        if (lane == 0) issued_s = i;
    } else {
        const int wq = warp & 3, et = threadIdx.x - 64;
        {
            // The scales of the CTA's k-blocks, all in flight together: those of the weights before the wait for the kernel in front, the
            // tokens' behind it; then the products.
            float* weights = scales + count * (HALVES * BT);                    // [64 rows each of gate and up, or one for all][k-block]
            auto copy4 = [](float* to, const float* from, bool in) {
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(gt_smem(to)), "l"(from), "r"(in ? 4 : 0) : "memory");
            };
            if (!p.early_w) pdl_wait();
            for (int k = et; k < count; k += 128) {
                copy4(weights + k, p.sw + (size_t)tb * p.ldsw + kb0 + k, true);
                if (GATED) copy4(weights + count + k, p.sw2 + (size_t)tb * p.ldsw2 + kb0 + k, true);
            }
            if (p.early_w) pdl_wait();
            for (int t = et >> 5; t < BT; t += 4) {                             // a warp takes a token, its lanes the k-blocks
                const bool in = t0 + t < p.M;
                const float* from = p.sx + (in ? (size_t)(t0 + t) * p.ldsx + kb0 : 0);
                for (int k = lane; k < count; k += 32) copy4(scales + k * (HALVES * BT) + t, from + (in ? k : 0), in);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("bar.sync 1, 128;" ::: "memory");
            for (int i = et; i < count * BT; i += 128) {
                const int k = i / BT, t = i % BT;
                const float x = scales[k * (HALVES * BT) + t];
                scales[k * (HALVES * BT) + t] = x * weights[k];
                if (GATED) scales[k * (HALVES * BT) + BT + t] = x * weights[count + k];
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
        }
        const uint32_t taddr = tmem_base + ((uint32_t)(wq * 32) << 16);
        const float* own_scales = scales + (GATED && wq >= 2 ? BT : 0);        // (lanes 64..127 hold up rows)
        uint64_t sums[BT / 2];
#pragma unroll
        for (int i = 0; i < BT / 2; ++i) sums[i] = 0;
        uint32_t turn = 0;
        for (int i = 0; i < count; ++i, ++turn) {
            const uint32_t slot = turn % S::SLOTS, use = turn / S::SLOTS;
            failed = ft_warp_failed(tfull0 + 8 * slot, use & 1, &abort_s, p);
            if (failed) break;
            tc_fence_after();
            const ulonglong2* sc = reinterpret_cast<const ulonglong2*>(own_scales + block_of(i) * (HALVES * BT));
#pragma unroll
            for (int c = 0; c < BT; c += 16) {
                uint32_t r[16];
                tc_ld16_nowait(taddr + slot * BT + c, r);
                ft_wait_ld(r);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const ulonglong2 s2 = sc[c / 4 + i];
                    ft_fma2(sums[c / 2 + 2 * i], r[4 * i], r[4 * i + 1], s2.x);
                    ft_fma2(sums[c / 2 + 2 * i + 1], r[4 * i + 2], r[4 * i + 3], s2.y);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty0 + 8 * slot);
        }
        // every load has landed and every product has read it: the stages' place takes the sums, [token][weight row]
        if (!abort_s) {
            float* to = reinterpret_cast<float*>(tiles) + wq * 32 + lane;
#pragma unroll
            for (int i = 0; i < BT / 2; ++i) {
                const float2 v = ft_floats(sums[i]);
                to[(2 * i) * S::LD] = v.x;
                to[(2 * i + 1) * S::LD] = v.y;
            }
        }
    }
    // (tensor memory goes back before the cluster's CTAs wait for one another, and the barrier says whether a warp gave up, see gemm_fp8_tc.cu)
    tc_fence_before();
    const bool gave_up = __syncthreads_or(failed);
    if (warp == 1) {
        if (gave_up) {
            ft_drain(full0, STAGES, asked_s);
            ft_drain(empty0, STAGES, issued_s);
        }
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(S::TMEM));
    }
    if (size > 1) cluster_sync_all();
    if (!gave_up)
        ft_emit<FT_ROWS, GATED, HALVES, 1, 8 / HALVES>(p, tiles_addr, S::LD, rank + size * warp, size * (FN_THREADS / 32), min(BT, p.M - t0), t0, tb);
    // (the peers may still read this CTA's sums)
    if (size > 1) cluster_sync_all();
}

template <int BT, bool GATED>
static int fn_launch(const CUtensorMap& mx, const CUtensorMap& mw, const CUtensorMap& mw2, Fp8TcParams& p, int splits, int sms, cudaStream_t stream) {
    using S = Fp8NarrowShape<BT>;
    constexpr int HALVES = GATED ? 2 : 1;
    p.tiles_m = (p.M + BT - 1) / BT;
    p.tiles_n = (p.N + FT_ROWS - 1) / FT_ROWS;
    splits = splits < 1 ? 1 : splits > 8 / HALVES ? 8 / HALVES : splits;
    if (splits > p.n_kb) splits = p.n_kb;
    p.kb_per_split = (p.n_kb + splits - 1) / splits;
    p.splits = (p.n_kb + p.kb_per_split - 1) / p.kb_per_split;
    const int size = p.splits * HALVES;
    const long long clusters = (long long)p.tiles_m * p.tiles_n, ctas = clusters * size;
    if (ctas > 0x7fffffff) return ACV_ERR_SIZE;
    // as many stages as the shared memory of an SM gives each of the CTAs that come to it (by the clusters that fit with one CTA to an SM)
    const int fixed = 1024 + 256 + (p.kb_per_split * HALVES * (BT + 1) * 4 + 127) / 128 * 128;
    const long long fit = (long long)ACV_CLUSTERS_AT_ONCE[size] * sms / 148 + 1;
    const int here = clusters < fit ? 1 : clusters < 2 * fit - 1 ? 2 : S::RESIDENT, budget = 227 * 1024 / here - 1024;
    if (fixed + S::SUMS > 225 * 1024 || fixed + 2 * S::STAGE > 225 * 1024) return ACV_ERR_SIZE;
    p.stages = (budget - fixed) / S::STAGE;
    p.stages = p.stages < 2 ? 2 : p.stages > 10 ? 10 : p.stages;            // (28 barriers at most in their 256 bytes)
    const int area = p.stages * S::STAGE > S::SUMS ? p.stages * S::STAGE : S::SUMS;
    auto kernel = gemm_fp8_narrow_kernel<BT, GATED>;
    static AcvSmemConfig cfg;
    if (const int rc = acv_ensure_smem(cfg, kernel, fixed + area)) return rc;
    acv_launch_cluster(PDL_GEMM, dim3(size, 1, 1), kernel, dim3((unsigned)ctas), dim3(FN_THREADS), fixed + area, stream, mx, mw, mw2, p);
    return acv_launch_status();
}

int acv_fp8_narrow(const CUtensorMap& mx, const CUtensorMap& mw, const CUtensorMap& mw2, Fp8TcParams& p, bool gated, int bt, int splits,
                   int sms, cudaStream_t stream) {
    switch (bt) {
        case 16: return gated ? fn_launch<16, true>(mx, mw, mw2, p, splits, sms, stream) : fn_launch<16, false>(mx, mw, mw2, p, splits, sms, stream);
        case 32: return gated ? fn_launch<32, true>(mx, mw, mw2, p, splits, sms, stream) : fn_launch<32, false>(mx, mw, mw2, p, splits, sms, stream);
        default: return ACV_ERR_SIZE;
    }
}
