// The products of e4m3 operands with block scales on the fifth-generation tensor cores.
//
//   y[t][n] = sum over groups g of 128 k of  sx[t][g] sw[n / 128][g] P_g[t][n],   P_g[t][n] = sum over k in g of qx[t][k] qw[n][k]
//
// P_g is what tcgen05.mma (kind::f8f6f4, operands staged by TMA, 128-byte swizzle: a k-block of 128 is one swizzle row) leaves in
// tensor memory for one k-block.  It cannot stay there: its scales differ from k-block to k-block.  Tensor memory holds several such
// partial tiles; while the tensor core fills one, the epilogue warps fetch another and add it, times its scales, to the float
// sums that they hold in registers (a fused multiply-add for each output and k-block, two at a time as fma.rn.f32x2).  Tokens are
// the rows (a lane holds one, so sx is a number of the thread's), features the columns, 64 to 128 of them to a thread.
//
// Two forms.  Pairs of CTAs on tiles of 256 x 256 or somewhat less (cta_group::2), persistent, for many tokens: a CTA loads 128 rows of each
// operand for a k-block, 32 KB for 512 cycles of tensor core.  And single CTAs on tiles of 128 x BN, one each, for fewer: K may be split over
// the CTAs of a cluster, whose sums meet through its shared memory, in rank order, so the result does not depend on timing.
//
// What bounds the many-token form beside the tensor core is that hand-over, once for each k-block: from the products' end until the
// epilogue warps of both CTAs have fetched the partial tile (some 500 cycles, the bandwidth of tensor memory) and the issuing warp has
// learnt it (as many), with two partial tiles for 512 cycles of tensor core each.  4096 x 4096 x 12288: 202 us; 143 us with nobody to wait for.
// Finer partial tiles, more epilogue warps or registers taken from the idle warps did not shorten it (four tiles of 128 columns 238 us,
// sixteen warps 310).
//
// Warps: 0 loads, 1 issues the products, from 2 on they are the epilogue, each a quarter of the lanes.  Every wait on an mbarrier is
// bounded; when one runs out the kernel records where in `status`, all roles leave their loops, the loads and products under way are
// waited for (with a limit, ft_drain), tensor memory is freed and the kernel returns.
#include "fp8_tc.cuh"

// sums[0 .. 8 PIECES) += scales * 16 PIECES columns of this lane's row, the first half of them from `first`, the others from `second`;
// a piece of sixteen is on its way while the one before is added.  Pieces from `change` on have the second scale.
template <int PIECES>
__device__ __forceinline__ void ft_add_tile(uint64_t* sums, uint32_t first, uint32_t second, float scale1, float scale2, int change = PIECES / 2) {
    const uint64_t s1 = ft_both(scale1), s2 = ft_both(scale2);
    uint32_t r[2][16];
    tc_ld16_nowait(first, r[0]);
    ft_wait_ld(r[0]);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        if (i + 1 < PIECES) tc_ld16_nowait(i + 1 < PIECES / 2 ? first + 16 * (i + 1) : second + 16 * (i + 1 - PIECES / 2), r[(i + 1) & 1]);
#pragma unroll
        for (int c = 0; c < 8; ++c) ft_fma2(sums[8 * i + c], r[i & 1][2 * c], r[i & 1][2 * c + 1], i < change ? s1 : s2);
        if (i + 1 < PIECES) ft_wait_ld(r[(i + 1) & 1]);
    }
}

// A row's scales, four k-blocks at a time and four ahead of their use: lanes hold rows, so a load looks 32 lines up whatever its width.
struct FtRowScales {
    const float* at;
    int left, vec;
    float now[4], next[4];
    __device__ __forceinline__ void fetch(float (&v)[4]) {
        if (vec && left >= 4) {
            const float4 f = *reinterpret_cast<const float4*>(at);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = i < left ? at[i] : 0.f;
        }
        at += 4;
        left -= 4;
    }
    __device__ __forceinline__ void begin(const float* row, int count, int aligned) {
        at = row;
        left = count;
        vec = aligned;
        fetch(now);
        fetch(next);
    }
    // the scale of the i-th k-block, i = 0, 1, 2, ...
    __device__ __forceinline__ float take(int i) {
        const float v = now[0];
        if ((i & 3) == 3) {
#pragma unroll
            for (int j = 0; j < 4; ++j) now[j] = next[j];
            fetch(next);
        } else {
            now[0] = now[1];
            now[1] = now[2];
            now[2] = now[3];
        }
        return v;
    }
};

// sixteen neighbouring outputs of a row
__device__ __forceinline__ void ft_store16(const Fp8TcParams& p, int row, int n, const uint64_t* v) {
    if (row >= p.M || n >= p.N) return;
    float f[16];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        const float2 t = ft_floats(v[c]);
        f[2 * c] = t.x;
        f[2 * c + 1] = t.y;
    }
    if (p.out_f32) {
        float* o = reinterpret_cast<float*>(p.out) + (size_t)row * p.ldo + n;
        if (p.out_vec && n + 16 <= p.N) {
#pragma unroll
            for (int c = 0; c < 4; ++c) reinterpret_cast<float4*>(o)[c] = make_float4(f[4 * c], f[4 * c + 1], f[4 * c + 2], f[4 * c + 3]);
        } else {
#pragma unroll
            for (int c = 0; c < 16; ++c)
                if (n + c < p.N) o[c] = f[c];
        }
    } else {
        bf16* o = reinterpret_cast<bf16*>(p.out) + (size_t)row * p.ldo + n;
        if (p.out_vec && n + 16 <= p.N) {
            uint32_t w[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) w[c] = pack_bf16x2(f[2 * c], f[2 * c + 1]);
            reinterpret_cast<uint4*>(o)[0] = make_uint4(w[0], w[1], w[2], w[3]);
            reinterpret_cast<uint4*>(o)[1] = make_uint4(w[4], w[5], w[6], w[7]);
        } else {
#pragma unroll
            for (int c = 0; c < 16; ++c)
                if (n + c < p.N) o[c] = __float2bfloat16_rn(f[c]);
        }
    }
}

__device__ __forceinline__ void ft_tile_of(int tile, int tiles_m, int tiles_n, int group, int& ta, int& tb) {
    const int per_group = group * tiles_n, g = tile / per_group, r = tile - g * per_group, rows = min(group, tiles_m - g * group);
    tb = r / rows;
    ta = g * group + (r - tb * rows);
}
// ----------------------------------------------------------------------------- pairs of CTAs, tiles of 256 x 256 and less
#define FP_STAGE (2 * FT_TILE)              // a CTA's share of a k-block: 128 rows of tokens, 128 of weights or less
#define FP_MAX_STAGES 6
#define FP_THREADS 320
#define FP_SLOTS 2                          // partial tiles in tensor memory

// The end of a pair of which a CTA gave up (both know it), by a warp of each.  One that stopped sooner asks for as many k-blocks as the other
// did (no more than the stages hold: a stage is asked for again only when both CTAs' loads of its last k-block have been used), so that the
// leader's barriers, which count both CTAs' loads, and with them the wait for what is under way come to their end.  What these loads
// bring is nobody's, so it is the matrices' first tile.
// (Nothing of this may cost the epilogue's loop registers, hence the numbers in shared memory; with the loop of loads unrolled tiles of 192
// columns spilled, 197 -> 231 us for 2048 tokens 5120 x 17408.)
struct FpEnd {
    uint32_t tiles;                     // where the stages are, the barriers behind them
    int asked, issued, other_asked;     // k-blocks whose loads and whose products are issued; the loads of the pair's other CTA
    int other_abort;
};
template <int COLS>
__device__ __forceinline__ void fp_settle(const volatile FpEnd& end, int stages, const CUtensorMap* map_x, const CUtensorMap* map_w) {
    const uint32_t tiles = end.tiles, full0 = tiles + stages * FP_STAGE;
    const int asked = max(end.asked, end.other_asked);
    const bool leads = cluster_ctarank() == 0;
#pragma unroll 1
    for (int i = end.asked; i < asked; ++i) {
        const uint32_t s = (uint32_t)i % (uint32_t)stages, stage = tiles + s * FP_STAGE, bar = cluster_map(full0 + 8 * s, 0);
        if (ft_elect()) {
            if (leads) mbar_expect_tx(full0 + 8 * s, 2 * (FT_TILE + COLS * FT_ROWS));
            tma_load_2d_pair(stage, map_x, bar, 0, 0);
            tma_load_2d_pair(stage + FT_TILE, map_w, bar, 0, 0);
        }
        __syncwarp();
    }
    if (leads) {
        ft_drain(full0, stages, asked);
        ft_drain(full0 + 8 * stages, stages, end.issued);
    }
}

// PIECES: a tile is 256 x 32 PIECES, an epilogue thread has 16 PIECES of its columns; where that is not 128, the thread's columns may lie in
// two blocks of the weights' scales.
// GATED: the tile's columns are 128 units' gate rows (the leader's half of the weight tile) and the same units' up rows (the other's).
template <bool GATED, int PIECES>
__global__ void __launch_bounds__(FP_THREADS, 1)
gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                     const __grid_constant__ CUtensorMap map_w2, const Fp8TcParams p) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* tiles = smem_raw + ((1024u - (gt_smem(smem_raw) & 1023u)) & 1023u);
    constexpr int COLS = 16 * PIECES, BYTES = 2 * (FT_TILE + COLS * FT_ROWS);       // of a thread or of a CTA's weight rows; of both CTAs' k-block
    const int STAGES = p.stages;
    const uint32_t tiles_addr = gt_smem(tiles);
    // barriers: full[STAGES] (the leader's count both CTAs' bytes), empty[STAGES], tmem_full[SLOTS], tmem_empty[SLOTS] (the leader's)
    const uint32_t full0 = tiles_addr + STAGES * FP_STAGE, empty0 = full0 + 8 * STAGES, tfull0 = empty0 + 8 * STAGES;
    const uint32_t tempty0 = tfull0 + 8 * FP_SLOTS;
    __shared__ uint32_t tmem_base_s;
    __shared__ volatile int abort_s;
    __shared__ volatile FpEnd end_s;
    __shared__ uint32_t most[GATED ? 2 : 1][2][FT_ROWS];
    __shared__ __align__(8) uint64_t met[4];            // the two warps of a quarter of the lanes tell each other their maxima
    const int warp = ft_warp(), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1, n_items = p.tiles_m * p.tiles_n;
    if (threadIdx.x == 0) {
        abort_s = 0;
        end_s.tiles = tiles_addr;
        end_s.asked = end_s.issued = end_s.other_abort = 0;
        for (int s = 0; s < STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int b = 0; b < FP_SLOTS; ++b) { mbar_init(tfull0 + 8 * b, 1); mbar_init(tempty0 + 8 * b, 16); }
        for (int q = 0; q < 4; ++q) mbar_init(gt_smem(&met[q]), 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(gt_smem(&tmem_base_s)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();         // both CTAs' barriers exist before a load or a commit of the other arrives at them
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_s;
    pdl_launch_dependents();

    if (warp == 0) {
        const uint32_t lead_full0 = cluster_map(full0, 0);
        const CUtensorMap* weights = GATED && rank == 1 ? &map_w2 : &map_w;
        auto load_w = [&](int s, int kb, int tb) {
            tma_load_2d_pair(tiles_addr + s * FP_STAGE + FT_TILE, weights, lead_full0 + 8 * s, kb * FT_ROWS,
                             GATED ? tb * FT_ROWS : (tb * 2 + (int)rank) * COLS);
        };
        int early = 0, asked = 0;
        if (p.early_w && pair < n_items) {
            int ta, tb;
            ft_tile_of(pair, p.tiles_m, p.tiles_n, p.group, ta, tb);
            early = min(STAGES, p.n_kb);
            if (ft_elect()) {
                for (int i = 0; i < early; ++i) {
                    if (rank == 0) mbar_expect_tx(full0 + 8 * i, BYTES);
                    load_w(i, i, tb);
                }
            }
            __syncwarp();
        }
        pdl_wait();
        int s = 0;
        uint32_t ph = 0;
        bool failed = false, ready = false;
        for (int item = pair; item < n_items && !failed; item += n_pairs) {
            int ta, tb;
            ft_tile_of(item, p.tiles_m, p.tiles_n, p.group, ta, tb);
            const int row = ta * 2 * FT_ROWS + (int)rank * FT_ROWS;
#pragma unroll 1
            for (int kb = 0; kb < p.n_kb; ++kb) {
                const bool half_done = asked < early;
                if (!half_done && !ready) {
                    failed = ft_warp_failed(empty0 + 8 * s, ph ^ 1, &abort_s, p, 1);
                    if (failed) break;
                }
                if (ft_elect()) {
                    if (!half_done && rank == 0) mbar_expect_tx(full0 + 8 * s, BYTES);
                    if (kb != p.skip_kb) {
                        tma_load_2d_pair(tiles_addr + s * FP_STAGE, &map_x, lead_full0 + 8 * s, kb * FT_ROWS, row);
                        if (!half_done) load_w(s, kb, tb);
                    }
                }
                __syncwarp();
                ++asked;
                if (++s == STAGES) { s = 0; ph ^= 1; }
                ready = __all_sync(0xffffffffu, ft_ready(empty0 + 8 * s, ph ^ 1));
            }
        }
        if (lane == 0) end_s.asked = asked;
    } else if (warp == 1) {
        if (rank == 0) {
            pdl_wait();         // (the first tokens come after it: the wait for them starts there)
            const uint32_t idesc = ft_idesc(2 * COLS, 2 * FT_ROWS);
            const uint64_t a0 = umma_desc(tiles_addr), b0 = umma_desc(tiles_addr + FT_TILE);
            uint32_t turn = 0, ph = 0;
            int s = 0;
            bool failed = false, ready = false;
            for (int item = pair; item < n_items && !failed; item += n_pairs) {
                for (int kb = 0; kb < p.n_kb; ++kb, ++turn) {
                    const uint32_t slot = turn % FP_SLOTS, use = turn / FP_SLOTS;
                    failed = (!ready && ft_warp_failed(full0 + 8 * s, ph, &abort_s, p, 3)) || ft_warp_failed(tempty0 + 8 * slot, (use & 1) ^ 1, &abort_s, p, 2);
                    if (failed) break;
                    tc_fence_after();
                    if (ft_elect()) {
                        const uint64_t a = a0 + (uint64_t)(s * (FP_STAGE >> 4)), b = b0 + (uint64_t)(s * (FP_STAGE >> 4));
                        const uint32_t d = tmem_base + slot * 2 * FT_ROWS;
#pragma unroll
                        for (int k = 0; k < 4; ++k) ft_mma<true>(d, a + 2 * k, b + 2 * k, idesc, k > 0);
                        tc_commit_pair(tfull0 + 8 * slot, 3);
                        tc_commit_pair(empty0 + 8 * s, 3);
                    }
                    __syncwarp();
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                    ready = __all_sync(0xffffffffu, ft_ready(full0 + 8 * s, ph));       // (the next k-block has landed)
                }
            }
            if (lane == 0) end_s.issued = (int)turn;
        }
    } else {
        const int wq = warp & 3, part = (warp - 2) >> 2;
        pdl_wait();
        const uint32_t lead_tempty0 = cluster_map(tempty0, 0);
        const uint32_t taddr = tmem_base + ((uint32_t)(wq * 32) << 16) + part * (GATED ? 64 : COLS);
        uint32_t turn = 0, parity = 0;
        // (a warp gives up as a whole: its loads from tensor memory and its exchanges are the whole warp's)
        bool failed = false;
        for (int item = pair; item < n_items && !failed; item += n_pairs) {
            int ta, tb;
            ft_tile_of(item, p.tiles_m, p.tiles_n, p.group, ta, tb);
            const int row = ta * 2 * FT_ROWS + (int)rank * FT_ROWS + wq * 32 + lane;
            // (rows and blocks that do not exist have products of zeros: any scale that does exist will do)
            const float* sx = p.sx + (size_t)min(row, p.M - 1) * p.ldsx;
            constexpr bool TWO = GATED || PIECES < 8;
            const int column = (tb * 2 + part) * COLS, last_block = (p.N - 1) / FT_ROWS, block = GATED ? tb : min(column / FT_ROWS, last_block);
            const int change = GATED || PIECES == 8 ? PIECES / 2 : (FT_ROWS - column % FT_ROWS) / 16;       // (the first piece of the next block)
            const float* sw = p.sw + (size_t)block * p.ldsw;
            const float* sw2 = GATED ? p.sw2 + (size_t)block * p.ldsw2 : p.sw + (size_t)min(block + 1, last_block) * p.ldsw;
            uint64_t sums[8 * PIECES];
#pragma unroll
            for (int i = 0; i < 8 * PIECES; ++i) sums[i] = 0;
            FtRowScales xs;
            xs.begin(sx, p.n_kb, p.sx_vec);
            float next_w = sw[0], next_w2 = TWO ? sw2[0] : 0.f;
            for (int kb = 0; kb < p.n_kb; ++kb, ++turn) {
                const float x = xs.take(kb), s1 = x * next_w, s2 = TWO ? x * next_w2 : s1;
                if (kb + 1 < p.n_kb) {
                    next_w = sw[kb + 1];
                    if (TWO) next_w2 = sw2[kb + 1];
                }
                const uint32_t slot = turn % FP_SLOTS, use = turn / FP_SLOTS;
                failed = ft_warp_failed(tfull0 + 8 * slot, use & 1, &abort_s, p);
                if (failed) break;
                tc_fence_after();
                const uint32_t t = taddr + slot * 2 * FT_ROWS;
                if (PIECES == 8) ft_add_tile<8>(sums, t, t + (GATED ? FT_ROWS : 64), s1, s2);
                else ft_add_tile<PIECES>(sums, t, t + PIECES / 2 * 16, s1, s2, change);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (rank == 0) mbar_arrive(tempty0 + 8 * slot);
                    else mbar_arrive_remote(lead_tempty0 + 8 * slot);
                }
            }
            if (failed) break;
            if (!GATED) {
#pragma unroll
                for (int i = 0; i < PIECES; ++i) ft_store16(p, row, column + 16 * i, sums + 8 * i);
            } else {
                // silu(gate) * up of 64 units, in the place of the gates' sums; the other 64 of the group are the partner warp's
                uint32_t m = 0;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float2 g = ft_floats(sums[i]), u = ft_floats(sums[32 + i]);
                    const float a = fp8_silu(g.x) * u.x, b = fp8_silu(g.y) * u.y;
                    m = max(m, max(fp8_magnitude(a), fp8_magnitude(b)));
                    sums[i] = ft_pair(a, b);
                }
                most[parity][part][wq * 32 + lane] = m;
                __syncwarp();
                if (lane == 0) mbar_arrive(gt_smem(&met[wq]));
                failed = ft_warp_failed(gt_smem(&met[wq]), parity, &abort_s, p);
                if (failed) break;
                const Fp8Scale k = fp8_scale(max(m, most[parity][part ^ 1][wq * 32 + lane]));
                parity ^= 1;
                if (row < p.M) {
                    if (part == 0) p.so[(size_t)row * p.ldso + tb] = k.s;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int u = tb * FT_ROWS + part * 64 + i * 16;
                        const uint64_t* v = sums + 8 * i;
                        uint8_t* o = reinterpret_cast<uint8_t*>(p.out) + (size_t)row * p.ldo + u;
                        uint32_t w[4];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float2 x = ft_floats(v[2 * c]), y = ft_floats(v[2 * c + 1]);
                            w[c] = fp8_pack4(x.x, x.y, y.x, y.y, k.r);
                        }
                        if (p.out_vec && u + 16 <= p.N) {
                            *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
                        } else {
#pragma unroll
                            for (int c = 0; c < 16; ++c)
                                if (u + c < p.N) o[c] = (uint8_t)(w[c >> 2] >> (8 * (c & 3)));
                        }
                    }
                }
            }
        }
    }
    // Neither CTA leaves, nor is the pair's tensor memory given back, while the other may still use this one's.  Each tells the other whether
    // it gave up and how many k-blocks it asked for: a barrier of the leader's counts both CTAs' loads.
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0) {
        ft_tell(cluster_map(gt_smem(const_cast<const int*>(&end_s.other_asked)), cluster_ctarank() ^ 1), end_s.asked);
        ft_tell(cluster_map(gt_smem(const_cast<const int*>(&end_s.other_abort)), cluster_ctarank() ^ 1), abort_s);
    }
    cluster_sync_all();
    if (abort_s | end_s.other_abort) {
        if (threadIdx.x < 32) fp_settle<COLS>(end_s, p.stages, &map_x, &map_w);
        cluster_sync_all();
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512));
    }
}

// ----------------------------------------------------------------------------- single CTAs, tiles of 128 x BN, K over a cluster
template <int BN>
struct Fp8TileShape {
    static constexpr int STAGE = FT_TILE + BN * FT_ROWS;
    static constexpr int SLOTS = BN <= 128 ? 4 : 2;                 // partial tiles in tensor memory
    static constexpr int TMEM = SLOTS * BN;
    static constexpr int LD = BN + 4;                               // floats of a row of the summed tile: sixteen-byte stores of eight rows meet no bank twice
    static constexpr int SUMS = FT_ROWS * LD * 4;
    static constexpr int COLS = BN / 2;                             // of an epilogue thread
    static constexpr int WARPS = 8;                                 // of the epilogue
    static constexpr int THREADS = 64 + 32 * WARPS;
    static constexpr int smem(int stages) { return 1024 + (stages * STAGE > SUMS ? stages * STAGE : SUMS) + 256; }
};

// GATED: BN is 256, the columns are 128 units' gate rows and their up rows, and a row of the result is a whole group.
template <int BN, bool GATED>
__global__ void __launch_bounds__(Fp8TileShape<BN>::THREADS, 1)
gemm_fp8_tile_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                     const __grid_constant__ CUtensorMap map_w2, const Fp8TcParams p) {
    using S = Fp8TileShape<BN>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* tiles = smem_raw + ((1024u - (gt_smem(smem_raw) & 1023u)) & 1023u);
    const int STAGES = p.stages;
    const uint32_t tiles_addr = gt_smem(tiles);
    const uint32_t full0 = tiles_addr + (STAGES * S::STAGE > S::SUMS ? STAGES * S::STAGE : S::SUMS), empty0 = full0 + 8 * STAGES;
    const uint32_t tfull0 = empty0 + 8 * STAGES, tempty0 = tfull0 + 8 * S::SLOTS;
    __shared__ uint32_t tmem_base_s;
    __shared__ volatile int abort_s;
    __shared__ int asked_s, issued_s;           // k-blocks whose loads and whose products are issued
    const int warp = ft_warp(), lane = threadIdx.x & 31;
    const int split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits, ta = tile % p.tiles_m, tb = tile / p.tiles_m;
    const int kb0 = split * p.kb_per_split, kb1 = min(kb0 + p.kb_per_split, p.n_kb);
    if (threadIdx.x == 0) {
        abort_s = 0;
        for (int s = 0; s < STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int b = 0; b < S::SLOTS; ++b) { mbar_init(tfull0 + 8 * b, 1); mbar_init(tempty0 + 8 * b, S::WARPS); }
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
    pdl_launch_dependents();
    const int row_here = ta * FT_ROWS;

    // Each column of tiles begins at another of its k-blocks (a multiple of four) and goes round: the CTAs, which start together, would
    // all read the same tokens' bytes at the same time (a tile's order is its own, whatever the others do).
    const int count = kb1 - kb0, turned = (int)(ft_spread(tb) % (unsigned)((count + 3) / 4)) * 4, wrap = count - turned;
    auto block_of = [&](int i) { return i < wrap ? i + turned : i - wrap; };
    bool failed = false;            // this warp gave up a wait
    if (warp == 0) {
        auto load_w = [&](int s, int kb) {
            const uint32_t dst = tiles_addr + s * S::STAGE + FT_TILE;
            if (GATED) {
                tma_load_2d(dst, &map_w, full0 + 8 * s, kb * FT_ROWS, tb * FT_ROWS);
                tma_load_2d(dst + FT_TILE, &map_w2, full0 + 8 * s, kb * FT_ROWS, tb * FT_ROWS);
            } else {
                tma_load_2d(dst, &map_w, full0 + 8 * s, kb * FT_ROWS, tb * BN);
            }
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
                    tma_load_2d(tiles_addr + s * S::STAGE, &map_x, full0 + 8 * s, kb * FT_ROWS, row_here);
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
        const uint32_t idesc = ft_idesc(BN, FT_ROWS);
        const uint64_t a0 = umma_desc(tiles_addr), b0 = umma_desc(tiles_addr + FT_TILE);
        uint32_t ph = 0;
        int s = 0;
        bool ready = false;
        int turn = 0;
        for (; turn < count; ++turn) {
            const uint32_t buf = (uint32_t)turn % S::SLOTS, use = (uint32_t)turn / S::SLOTS;
            if ((!ready && ft_warp_failed(full0 + 8 * s, ph, &abort_s, p, 3)) ||
                (use && ft_warp_failed(tempty0 + 8 * buf, (use & 1) ^ 1, &abort_s, p, 2)))
                break;
            tc_fence_after();
            if (ft_elect()) {
                const uint64_t a = a0 + (uint64_t)(s * (S::STAGE >> 4)), b = b0 + (uint64_t)(s * (S::STAGE >> 4));
                const uint32_t d = tmem_base + buf * BN;
#pragma unroll
                for (int k = 0; k < 4; ++k) ft_mma<false>(d, a + 2 * k, b + 2 * k, idesc, k > 0);
                tc_commit(tfull0 + 8 * buf);
                tc_commit(empty0 + 8 * s);
            }
            __syncwarp();
            if (++s == STAGES) { s = 0; ph ^= 1; }
            ready = __all_sync(0xffffffffu, ft_ready(full0 + 8 * s, ph));
        }
        failed = turn < count;
        if (lane == 0) issued_s = turn;
    } else {
        const int wq = warp & 3, part = (warp - 2) >> 2;
        pdl_wait();
        const uint32_t taddr = tmem_base + ((uint32_t)(wq * 32) << 16);
        const int r = wq * 32 + lane;
        const float* sx = p.sx + (size_t)min(row_here + r, p.M - 1) * p.ldsx;
        const int block = GATED ? tb : min(tb * BN / FT_ROWS, (p.N - 1) / FT_ROWS);
        const float *sw = p.sw + (size_t)block * p.ldsw + kb0, *sw2 = GATED ? p.sw2 + (size_t)block * p.ldsw2 + kb0 : nullptr;
        uint64_t sums[S::COLS / 2];
#pragma unroll
        for (int i = 0; i < S::COLS / 2; ++i) sums[i] = 0;
        FtRowScales xs;
        xs.begin(sx + kb0 + turned, wrap, p.sx_vec && !(kb0 & 3));
        float next_w = sw[turned], next_w2 = GATED ? sw2[turned] : 0.f;
        for (int turn = 0; turn < count; ++turn) {
            if (turn == wrap) xs.begin(sx + kb0, turned, p.sx_vec && !(kb0 & 3));
            const float x = xs.take(turn < wrap ? turn : turn - wrap), s1 = x * next_w, s2 = GATED ? x * next_w2 : s1;
            if (turn + 1 < count) {
                next_w = sw[block_of(turn + 1)];
                if (GATED) next_w2 = sw2[block_of(turn + 1)];
            }
            const uint32_t buf = (uint32_t)turn % S::SLOTS, use = (uint32_t)turn / S::SLOTS;
            failed = ft_warp_failed(tfull0 + 8 * buf, use & 1, &abort_s, p);
            if (failed) break;
            tc_fence_after();
            const uint32_t t = taddr + buf * BN;
            if (GATED) ft_add_tile<S::COLS / 16>(sums, t + part * 64, t + FT_ROWS + part * 64, s1, s2);
            else ft_add_tile<S::COLS / 16>(sums, t + part * 64, t + part * 64 + 32, s1, s1);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(tempty0 + 8 * buf);
        }
        // Every load has landed and every product has read it: the stages' place takes the tile's sums, [row][column].  (After a wait
        // that ran out neither is sure, and nothing is written.)
        if (!abort_s && row_here + r < p.M) {
            float* to = reinterpret_cast<float*>(tiles) + r * S::LD;
#pragma unroll
            for (int i = 0; i < S::COLS / 4; ++i) {
                const float2 lo = ft_floats(sums[2 * i]), hi = ft_floats(sums[2 * i + 1]);
                const int c = i < 16 ? part * 64 + 4 * i : FT_ROWS + part * 64 + 4 * (i - 16);      // (the second 64: the up rows')
                *reinterpret_cast<float4*>(to + c) = make_float4(lo.x, lo.y, hi.x, hi.y);
            }
        }
    }
    // Tensor memory goes back before the cluster's CTAs wait for one another: a CTA that held some while it waited for a peer, which waits for
    // some that another kernel's CTA holds in the same way, would wait for good.
    // (Whether a warp gave up comes with the barrier: a look at the flag behind it took 0.05 us of every kernel's end.)
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
    if (p.splits > 1) cluster_sync_all();
    if (!gave_up) {
        const int first = split + p.splits * warp, step = p.splits * (S::THREADS / 32), rows = min(FT_ROWS, p.M - row_here);
        if (p.splits == 1) ft_emit<BN, GATED, 1, 4, 1>(p, tiles_addr, S::LD, first, step, rows, row_here, tb);
        else if (p.splits <= 4 && rows > 2 * step) ft_emit<BN, GATED, 1, 4, 4>(p, tiles_addr, S::LD, first, step, rows, row_here, tb);
        else if (rows <= step) ft_emit<BN, GATED, 1, 1, 8>(p, tiles_addr, S::LD, first, step, rows, row_here, tb);
        else ft_emit<BN, GATED, 1, 2, 8>(p, tiles_addr, S::LD, first, step, rows, row_here, tb);
    }
    // (the peers may still read this CTA's sums)
    if (p.splits > 1) cluster_sync_all();
}

// ----------------------------------------------------------------------------- host side
// Test of the bounded waits, without a fault: the next product launched from this process polls each mbarrier at most `wait_limit`
// times and its producer leaves out the loads of k-block `skip_kb` (the codes are those of acv_gemm_tc_test_fault; the output of that
// launch is unspecified).
static unsigned int g_test_wait_limit = 0;
static int g_test_skip_kb = -1;
ACV_API void acv_gemm_fp8_test_fault(int wait_limit, int skip_kb) {
    g_test_wait_limit = wait_limit > 0 ? (unsigned int)wait_limit : 0u;
    g_test_skip_kb = skip_kb;
}

template <bool GATED, int PIECES>
static int ft_launch_pair(const CUtensorMap& mx, const CUtensorMap& mw, const CUtensorMap& mw2, Fp8TcParams& p, int sms, cudaStream_t stream) {
    p.stages = FP_MAX_STAGES;
    const int smem = FP_MAX_STAGES * FP_STAGE + 1024 + 256;
    auto kernel = gemm_fp8_pair_kernel<GATED, PIECES>;
    static AcvSmemConfig cfg;
    if (const int rc = acv_ensure_smem(cfg, kernel, smem)) return rc;
    // pairs that can be resident at once: two free SMs side by side each, which an odd number of SMs in a part of the chip does not give
    static std::mutex mu;
    static int pairs_of_device[64];
    int dev = 0, resident = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return ACV_ERR_SIZE;
    {
        std::lock_guard<std::mutex> lock(mu);
        resident = pairs_of_device[dev];
        if (resident <= 0) {
            cudaLaunchConfig_t lc = {};
            lc.gridDim = dim3(2 * (sms / 2));
            lc.blockDim = dim3(FP_THREADS);
            lc.dynamicSmemBytes = smem;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
            lc.attrs = attr;
            lc.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&resident, kernel, &lc) != cudaSuccess || resident <= 0) {
                cudaGetLastError();
                return ACV_ERR_SIZE;
            }
            pairs_of_device[dev] = resident;
        }
    }
    p.tiles_m = (p.M + 2 * FT_ROWS - 1) / (2 * FT_ROWS);
    const int wide = GATED ? FT_ROWS : 32 * PIECES;
    p.tiles_n = (p.N + wide - 1) / wide;
    p.group = 8;
    const long long items = (long long)p.tiles_m * p.tiles_n;
    if (items > 0x7fffffff) return ACV_ERR_SIZE;
    const int pairs = (int)(items < resident ? items : resident);
    acv_launch_cluster(PDL_GEMM, dim3(2, 1, 1), kernel, dim3(2 * pairs), dim3(FP_THREADS), smem, stream, mx, mw, mw2, p);
    return acv_launch_status();
}

template <int BN, bool GATED>
static int ft_launch_tile(const CUtensorMap& mx, const CUtensorMap& mw, const CUtensorMap& mw2, Fp8TcParams& p, int splits, cudaStream_t stream) {
    using S = Fp8TileShape<BN>;
    p.tiles_m = (p.M + FT_ROWS - 1) / FT_ROWS;
    p.tiles_n = (p.N + (GATED ? FT_ROWS : BN) - 1) / (GATED ? FT_ROWS : BN);
    if (splits < 1) splits = 1;
    if (splits > 8) splits = 8;
    if (splits > p.n_kb) splits = p.n_kb;
    p.kb_per_split = (p.n_kb + splits - 1) / splits;
    p.splits = (p.n_kb + p.kb_per_split - 1) / p.kb_per_split;
    p.stages = min(8, 200 * 1024 / S::STAGE);
    const int smem = S::smem(p.stages);
    auto kernel = gemm_fp8_tile_kernel<BN, GATED>;
    static AcvSmemConfig cfg;
    if (const int rc = acv_ensure_smem(cfg, kernel, smem)) return rc;
    const long long ctas = (long long)p.tiles_m * p.tiles_n * p.splits;
    if (ctas > 0x7fffffff) return ACV_ERR_SIZE;
    acv_launch_cluster(PDL_GEMM, dim3(p.splits, 1, 1), kernel, dim3((unsigned)ctas), dim3(S::THREADS), smem, stream, mx, mw, mw2, p);
    return acv_launch_status();
}

// (Microseconds of calls in bursts, before the board's power cap is felt.)  How a product is made: kind 1 the streaming kernel (gemm_fp8_rows.cu), 2 tiles of 128 x bn with K over `splits` CTAs, 3 pairs on tiles of 256 x bn, 4 weight
// rows on the tensor core's rows, bn tokens to a tile, K over `splits` CTAs (gemm_fp8_narrow.cu).
//
// Up to 16 tokens whose weights are one round of blocks of 32 rows stream (microseconds, streaming and the best of kind 4: 8 tokens
// 4096 x 4096 4.2, 5.4; 6144 x 4096 7.6, 5.8; 4096 x 12288 11.6, 11.2; 16 tokens 4096 x 2560 4.6, 4.9; 1024 x 4096 5.4, 4.1).
// Up to 32 tokens, and beyond: kind 4 and kind 2, 32 tokens 6144 x 4096 7.2 and 12.7, 64 tokens 6144 x 4096 11.2 and 9.9,
// 4096 x 12288 15.9 and 14.0, 5120 x 17408 20.8 and 20.8.
//   Splits of K are what fits the SMs at once in clusters, two CTAs of kind 4 to an SM (three of the gated form, whose cluster holds two
// halves of a group), one of kind 2, and at least four k-blocks to each: 16 tokens 6144 x 4096 in 2, 4, 6 splits 7.9, 6.1, 9.8; 4096 x 1024
// in 1, 2, 4: 4.3, 3.8, 4.2; 12288 units, K 4096, in 1, 2, 3: 21.0, 19.2, 24.8 (the gated form stays with two: where few units leave SMs idle
// four would be faster, 32 tokens, 1361 units of 11216 in 2 and 4: 18, 12; 3000 units of 4096: 10.3, 9.5); kind 2, 65 tokens 4096 x 12288 in 2, 3, 4, 6: 19.5, 15.9,
// 14.0, 23.3.  Kind 4 holds the scales of its k-blocks in shared memory beside its stages: 160 KB of them at most, about 80 thousand k to a
// split of 32 tokens' gated form, and longer rows are kind 2's (one that holds none).
//   Pairs of CTAs and tiles of 128 rows both come in rounds over the SMs.  A round of pairs takes 1.5 of a round of tiles of 128 x 128
// (1024 tokens 5120 x 17408 in 2 and 3: 143 us and 136; 6144 x 4096, 512 tokens in 1 and 2: 28, 32; 2048 in 3 and 6: 63, 82), 0.83 of
// one of gated tiles of 128 x 256 (12288 units of 4096, 256 tokens in 2 and 2: 43.8, 50.1; 384 in 3 and 2: 69, 54), and K over several CTAs brings a
// round of those down with it (100 tokens of 8704 units of 5120, pairs and 2 splits: 31, 26; 39 of 1361 units of 11216, pairs and 8: 49, 13).  Pairs take tiles of
// 256 columns, or of 224 or 192 where those come in few enough rounds: such a round takes 0.94 and 0.87 (with 256, 224 and 192 columns, 1024
// tokens 7168 x 5120 in 2, 2, 3 rounds 49.7, 46.1, 57.4; 5120 x 17408 in 2, 2, 2: 143, 135, 122; 4096 tokens 4096 x 12288 in 4, 5, 5: 202, 257, 234).
struct Fp8Plan { int kind, bn, splits; };
static Fp8Plan ft_plan(int M, int N, int K, bool gated, int sms) {
    const long long n_kb = (K + FT_ROWS - 1) / FT_ROWS, wide = (N + FT_ROWS - 1) / FT_ROWS, deep = (M + FT_ROWS - 1) / FT_ROWS;
    auto fit = [&](int size) { return (long long)ACV_CLUSTERS_AT_ONCE[size] * sms / 148; };
    if (!gated && M <= 16 && N <= 32ll * sms && K <= (M <= 8 ? 8192 : 2560)) return {1, 0, 1};
    int splits = 1;
    if (M <= 32) {
        if (gated) splits = wide <= 3 * fit(4) && n_kb >= 4 ? 2 : 1;
        else
            while (splits < 8 && wide <= 2 * fit(splits + 1) && n_kb >= 4 * (splits + 1)) ++splits;
        const int bt = M <= 16 ? 16 : 32;
        if ((n_kb + splits - 1) / splits * (gated ? 2 : 1) * (bt + 1) * 4 <= 160 * 1024) return {4, bt, splits};
        splits = 1;
    }
    const long long tiles = deep * wide, tile_rounds = (tiles + sms - 1) / sms;
    auto rounds_of = [&](long long across) { return (double)(((deep + 1) / 2 * across + sms / 2 - 1) / (sms / 2)); };
    while (splits < 8 && tiles <= fit(splits + 1) && n_kb >= 4 * (splits + 1)) ++splits;
    if (gated) {
        if (rounds_of(wide) * 0.83 < (splits > 1 ? 1. / splits + 0.25 : (double)tile_rounds)) return {3, 256, 1};
    } else {
        const double by256 = rounds_of((wide + 1) / 2), by224 = rounds_of((N + 223) / 224) * 0.94, by192 = rounds_of((N + 191) / 192) * 0.87;
        const double least = min(by256, min(by224, by192));
        if (least * 1.5 < (double)tile_rounds) return {3, by256 <= least ? 256 : by224 <= least ? 224 : 192, 1};
    }
    return {2, gated ? 256 : 128, splits};
}

static int ft_run(Fp8Operands& o, int flags, int plan, int* status, int sms, cudaStream_t stream) {
    const bool gated = o.w2 != nullptr;
    if (o.M <= 0 || o.N <= 0) return 0;
    if (o.K <= 0 || max(o.M, max(o.N, o.K)) > 0x7fffffff - 1024) return ACV_ERR_SIZE;       // (sizes are rounded up to tiles in 32 bits)
    // a single row's stride says nothing; several rows do not overlap
    const long long row_bytes = ((long long)o.K + 15) / 16 * 16;
    if (o.M == 1) o.ldx = row_bytes;
    if (o.N == 1) { o.ldw = row_bytes; if (gated) o.ldw2 = row_bytes; }
    if (o.ldx < o.K || o.ldw < o.K || (gated && o.ldw2 < o.K)) return ACV_ERR_ALIGN;
    if (((uintptr_t)o.x | (uintptr_t)o.w | (uintptr_t)o.w2) % 16 || (o.ldx | o.ldw | o.ldw2) % 16) return ACV_ERR_ALIGN;
    const Fp8Plan how = plan ? Fp8Plan{plan & 15, (plan >> 4) & 0xfff, plan >> 16} : ft_plan(o.M, o.N, o.K, gated, sms);
    if (how.kind == 1) return acv_fp8_rows(o, flags, stream);
    if (!status) return ACV_ERR_SCRATCH;
    Fp8TcParams p = {};
    p.M = o.M; p.N = o.N; p.n_kb = (o.K + FT_ROWS - 1) / FT_ROWS;
    p.sx = o.sx; p.sw = o.sw; p.sw2 = o.sw2; p.ldsx = o.ldsx; p.ldsw = o.ldsw; p.ldsw2 = o.ldsw2; p.ldo = o.ldo; p.ldso = o.ldso;
    p.out = o.out; p.so = o.so; p.out_f32 = o.out_f32; p.early_w = flags & 1; p.status = status;
    p.out_vec = fp8_rows_aligned(o.out, o.ldo, gated ? 1 : o.out_f32 ? 4 : 2, 16);
    p.sx_vec = fp8_rows_aligned(o.sx, o.ldsx, 4, 16);
    p.wait_limit = g_test_wait_limit ? g_test_wait_limit : GT_WAIT_LIMIT;
    p.skip_kb = g_test_skip_kb;
    g_test_wait_limit = 0; g_test_skip_kb = -1;
    CUtensorMap mx, mw, mw2;
    if (how.kind == 4 && how.bn != 16 && how.bn != 32) return ACV_ERR_SIZE;
    if (how.kind == 2 && how.bn != (gated ? 256 : 128)) return ACV_ERR_SIZE;
    if (const int rc = ft_map(&mx, o.x, o.M, o.K, o.ldx, how.kind == 4 ? how.bn : FT_ROWS)) return rc;
    if (how.kind == 3 && how.bn != 256 && (gated || (how.bn != 224 && how.bn != 192))) return ACV_ERR_SIZE;
    if (const int rc = ft_map(&mw, o.w, o.N, o.K, o.ldw, how.kind == 4 && gated ? 64 : how.kind == 3 ? how.bn / 2 : FT_ROWS)) return rc;
    mw2 = mw;
    if (gated)
        if (const int rc = ft_map(&mw2, o.w2, o.N, o.K, o.ldw2, how.kind == 4 ? 64 : FT_ROWS)) return rc;
    if (how.kind == 3) {
        if (gated) return ft_launch_pair<true, 8>(mx, mw, mw2, p, sms, stream);
        return how.bn == 256   ? ft_launch_pair<false, 8>(mx, mw, mw2, p, sms, stream)
               : how.bn == 224 ? ft_launch_pair<false, 7>(mx, mw, mw2, p, sms, stream)
                               : ft_launch_pair<false, 6>(mx, mw, mw2, p, sms, stream);
    }
    if (how.kind == 4) return acv_fp8_narrow(mx, mw, mw2, p, gated, how.bn, how.splits, sms, stream);
    if (how.kind != 2) return ACV_ERR_SIZE;
    return gated ? ft_launch_tile<256, true>(mx, mw, mw2, p, how.splits, stream) : ft_launch_tile<128, false>(mx, mw, mw2, p, how.splits, stream);
}

// A call's arguments as one record (a caller through a foreign-function interface pays for each argument by itself), field for field as
// kernels/ops.py packs them.  x [M,K] bytes, sx [M][groups of K]; w [N,K] bytes, sw [blocks of N][groups of K]; out [M,N] float or
// bfloat16; every matrix's rows at a stride of its own, those of x and w on 16 bytes.  With w2, sw2 and so, the gated form: w and w2 are
// gate and up rows, out [M,N] bytes = silu(gate) * up by its own scales so [M][groups of N].  flags: 1 the weights were written
// long before, they may be read while the kernel in front still runs.  plan: 0, or kind | bn << 4 | splits << 16.  status: one int,
// 0 unless a bounded wait ran out.
struct Fp8LinearArgs {
    const void *x, *sx, *w, *sw, *out, *w2, *sw2, *so, *status, *stream;
    long long ldx, ldsx, ldw, ldsw, ldo, ldw2, ldsw2, ldso;
    int M, N, K, out_f32, flags, plan, sms;
};
ACV_API int acv_linear_fp8(const Fp8LinearArgs* a) {
    Fp8Operands o = {};
    o.x = (const uint8_t*)a->x; o.w = (const uint8_t*)a->w; o.w2 = (const uint8_t*)a->w2;
    o.sx = (const float*)a->sx; o.sw = (const float*)a->sw; o.sw2 = (const float*)a->sw2;
    o.out = const_cast<void*>(a->out); o.so = (float*)const_cast<void*>(a->so);
    o.ldx = a->ldx; o.ldw = a->ldw; o.ldw2 = a->ldw2; o.ldo = a->ldo; o.ldsx = a->ldsx; o.ldsw = a->ldsw; o.ldsw2 = a->ldsw2; o.ldso = a->ldso;
    o.M = a->M; o.N = a->N; o.K = a->K; o.out_f32 = a->out_f32;
    if (o.w2 && (!o.sw2 || !o.so)) return ACV_ERR_SIZE;
    return ft_run(o, a->flags, a->plan, (int*)const_cast<void*>(a->status), a->sms, (cudaStream_t)const_cast<void*>(a->stream));
}
