// The products of e4m3 operands with block scales for a few tokens: every weight is read once, which is what bounds them.
//
//   y[t][n] = sum over groups g of 128 k of  sx[t][g] sw[n / 128][g] sum over k in g of qx[t][k] qw[n][k]
//
// A group's inner sum is four mma.sync of 32 k (weight rows are its M, tokens its N) into float; the two scales multiply it as it
// joins the running float sum.  As in gemm_rows.cu a lane brings its own operands by 16-byte asynchronous copies into a ring that it
// alone reads, so no barrier stands in the loop: a group of a row is 128 bytes, as 64 bfloat16 are, and the ring's layout is the same.
// Which k of a group a lane holds is the same for tokens and weights.
#include "fp8.cuh"
#include "gemm_fp8.h"
#include "rows_ring.cuh"

struct Fp8RowsParams : Fp8Operands {
    int G, early_w;                     // groups of K; the weights may be read before the kernel in front has ended
};

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// sixteen bytes of a row at k, of which those behind K are zeros (`in` false: all of them)
__device__ __forceinline__ void copy16_of_row(uint32_t dst, const uint8_t* row, int k, int K, bool in) {
    const int n = in ? max(0, min(16, K - k)) : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(n > 0 ? row + k : row), "r"(n));
}

// total[a][h] += scales * (the group's sums of sixteen rows and eight tokens)
template <int R, int H>
__device__ __forceinline__ void fp8_add_group(const RrChunk<R, H>& k, float (&total)[R / 2][H][4], const float* sx, float sw0, float sw1) {
#pragma unroll
    for (int a = 0; a < R / 2; ++a)
#pragma unroll
        for (int h = 0; h < H; ++h) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const uint4 lo = k.w[b][2 * a], hi = k.w[b][2 * a + 1], x = k.x[b][h];
                mma_e4m3(c, lo.x, hi.x, lo.y, hi.y, x.x, x.y);
                mma_e4m3(c, lo.z, hi.z, lo.w, hi.w, x.z, x.w);
            }
            const float s0 = sx[8 * h], s1 = sx[8 * h + 1];
            total[a][h][0] = fmaf(c[0], s0 * sw0, total[a][h][0]);
            total[a][h][1] = fmaf(c[1], s1 * sw0, total[a][h][1]);
            total[a][h][2] = fmaf(c[2], s0 * sw1, total[a][h][2]);
            total[a][h][3] = fmaf(c[3], s1 * sw1, total[a][h][3]);
        }
}

// A block takes 8 R weight rows at a time and its eight warps an eighth of the groups each; R: 2 or 4, H: octets of tokens, DEPTH:
// groups in a warp's ring.  The tokens' scales of a warp's groups are fetched once, into shared memory of its own.
template <int R, int H, int DEPTH>
__global__ void __launch_bounds__(RR_WARPS * 32, 2) gemm_fp8_rows_kernel(const Fp8RowsParams p) {
    using Chunk = RrChunk<R, H>;
    constexpr int CHUNK = Chunk::BYTES, COLS = 8 * R;
    extern __shared__ __align__(16) unsigned char ring[];
    __shared__ float part[2][RR_WARPS][8 * H][COLS + 4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
    const int tiles = (p.N + COLS - 1) / COLS, t0 = blockIdx.y * 8 * H;
    const int c0 = p.G * warp / RR_WARPS, chunks = p.G * (warp + 1) / RR_WARPS - c0;
    const uint32_t own = smem_u32(ring) + warp * (DEPTH * CHUNK) + lane * 16;
    float* sx = reinterpret_cast<float*>(ring + RR_WARPS * DEPTH * CHUNK) + (size_t)c0 * 8 * H;      // [its groups][8 H tokens]
    int w_tile = blockIdx.x, w_next = 0, w_into = 0, x_tile = blockIdx.x, x_next = 0, x_into = 0;
    auto ask_w = [&]() {
        if (w_tile >= tiles) return;
        const uint32_t dst = own + w_into * CHUNK;
        const int k = (c0 + w_next) * FP8_GROUP + tq * 16;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = w_tile * COLS + r * 8 + g;
            const uint8_t* src = p.w + (size_t)min(row, p.N - 1) * p.ldw;
#pragma unroll
            for (int b = 0; b < 2; ++b) copy16_of_row(Chunk::weights_at(dst, b, r), src, k + b * 64, p.K, row < p.N);
        }
        w_into = w_into + 1 == DEPTH ? 0 : w_into + 1;
        if (++w_next == chunks) { w_next = 0; w_tile += gridDim.x; }
    };
    auto ask_x = [&]() {
        if (x_tile < tiles) {
            const uint32_t dst = own + x_into * CHUNK;
            const int k = (c0 + x_next) * FP8_GROUP + tq * 16;
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const int t = t0 + h * 8 + g;
                const uint8_t* src = p.x + (size_t)min(t, p.M - 1) * p.ldx;
#pragma unroll
                for (int b = 0; b < 2; ++b) copy16_of_row(Chunk::tokens_at(dst, b, h), src, k + b * 64, p.K, t < p.M);
            }
            x_into = x_into + 1 == DEPTH ? 0 : x_into + 1;
            if (++x_next == chunks) { x_next = 0; x_tile += gridDim.x; }
        }
        cp_async_commit();
    };
    if (p.early_w && chunks) {
#pragma unroll
        for (int i = 0; i < DEPTH - 1; ++i) ask_w();
    }
    pdl_launch_dependents();
    pdl_wait();
    if (chunks) {
#pragma unroll
        for (int i = 0; i < DEPTH - 1; ++i) {
            if (!p.early_w) ask_w();
            ask_x();
        }
        for (int i = lane; i < chunks * 8 * H; i += 32) {
            const int t = t0 + i % (8 * H);
            sx[i] = t < p.M ? p.sx[t * p.ldsx + c0 + i / (8 * H)] : 0.f;
        }
        __syncwarp();
    }
    int from = 0;
    for (int tile = blockIdx.x, turn = 0; tile < tiles; tile += gridDim.x, turn ^= 1) {
        float total[R / 2][H][4];
#pragma unroll
        for (int a = 0; a < R / 2; ++a)
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) total[a][h][i] = 0.f;
        const float* sw = p.sw + (size_t)(tile * COLS / FP8_GROUP) * p.ldsw + c0;
        float scale = chunks ? __ldg(sw) : 0.f;
#pragma unroll 1
        for (int n = 0; n < chunks; ++n) {
            const float s = scale;
            if (n + 1 < chunks) scale = __ldg(sw + n + 1);
            cp_async_wait<DEPTH - 2>();
            const uint32_t src = own + from * CHUNK;
            from = from + 1 == DEPTH ? 0 : from + 1;
            Chunk chunk;
            chunk.read(src);
            ask_w();
            ask_x();
            fp8_add_group<R, H>(chunk, total, sx + n * 8 * H + 2 * tq, s, s);
        }
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < 2; ++e) part[turn][warp][h * 8 + 2 * tq + e][r * 8 + g] = total[r / 2][h][2 * (r & 1) + e];
        __syncthreads();
        for (int i = threadIdx.x; i < 8 * H * COLS; i += RR_WARPS * 32) {
            const int m = i / COLS, q = i - m * COLS, t = t0 + m, n = tile * COLS + q;
            if (t >= p.M || n >= p.N) continue;
            const float v = rr_sum(part[turn], m, q);
            if (p.out_f32) reinterpret_cast<float*>(p.out)[t * p.ldo + n] = v;
            else reinterpret_cast<bf16*>(p.out)[t * p.ldo + n] = __float2bfloat16_rn(v);
        }
    }
    cp_async_wait<0>();
}

// The gated form, silu(gate) * up quantised for the next product.  A warp takes eight units: their gate rows are rows 0..7 of its
// sixteen, their up rows 8..15, so a lane holds both sums of a unit and a token.  Four warps are a block (32 units), four blocks a
// cluster: a group of 128 units, whose maximum travels through the cluster's shared memory before the group is written.
#define FG_WARPS 4
template <int H, int DEPTH>
__global__ void __launch_bounds__(FG_WARPS * 32) gemm_fp8_rows_gated_kernel(const Fp8RowsParams p) {
    using Chunk = RrChunk<2, H>;
    constexpr int CHUNK = Chunk::BYTES;
    extern __shared__ __align__(16) unsigned char ring[];
    __shared__ uint32_t most[FG_WARPS * 4][8 * H];         // the largest magnitude of each warp of the cluster and each token
    __shared__ uint8_t codes[8 * H][FG_WARPS * 8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
    const int t0 = blockIdx.y * 8 * H, u0 = blockIdx.x * (FG_WARPS * 8), unit = u0 + warp * 8 + g;
    const uint32_t own = smem_u32(ring) + warp * (DEPTH * CHUNK) + lane * 16;
    float* sx = reinterpret_cast<float*>(ring + FG_WARPS * DEPTH * CHUNK);                  // [groups][8 H tokens]
    const uint8_t* wg = p.w + (size_t)min(unit, p.N - 1) * p.ldw;
    const uint8_t* wu = p.w2 + (size_t)min(unit, p.N - 1) * p.ldw2;
    int w_next = 0, w_into = 0, x_next = 0, x_into = 0;
    auto ask_w = [&]() {
        if (w_next >= p.G) return;
        const uint32_t dst = own + w_into * CHUNK;
        const int k = w_next * FP8_GROUP + tq * 16;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            copy16_of_row(Chunk::weights_at(dst, b, 0), wg, k + b * 64, p.K, unit < p.N);
            copy16_of_row(Chunk::weights_at(dst, b, 1), wu, k + b * 64, p.K, unit < p.N);
        }
        w_into = w_into + 1 == DEPTH ? 0 : w_into + 1;
        ++w_next;
    };
    auto ask_x = [&]() {
        if (x_next < p.G) {
            const uint32_t dst = own + x_into * CHUNK;
            const int k = x_next * FP8_GROUP + tq * 16;
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const int t = t0 + h * 8 + g;
                const uint8_t* src = p.x + (size_t)min(t, p.M - 1) * p.ldx;
#pragma unroll
                for (int b = 0; b < 2; ++b) copy16_of_row(Chunk::tokens_at(dst, b, h), src, k + b * 64, p.K, t < p.M);
            }
            x_into = x_into + 1 == DEPTH ? 0 : x_into + 1;
            ++x_next;
        }
        cp_async_commit();
    };
    if (p.early_w) {
#pragma unroll
        for (int i = 0; i < DEPTH - 1; ++i) ask_w();
    }
    cluster_arrive();           // (waited for before the first word to a peer)
    pdl_launch_dependents();
    pdl_wait();
#pragma unroll
    for (int i = 0; i < DEPTH - 1; ++i) {
        if (!p.early_w) ask_w();
        ask_x();
    }
    for (int i = threadIdx.x; i < p.G * 8 * H; i += FG_WARPS * 32) {
        const int t = t0 + i % (8 * H);
        sx[i] = t < p.M ? p.sx[t * p.ldsx + i / (8 * H)] : 0.f;
    }
    __syncthreads();
    float total[1][H][4];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) total[0][h][i] = 0.f;
    const int block_row = min(u0, p.N - 1) / FP8_GROUP;
    const float *sg = p.sw + (size_t)block_row * p.ldsw, *su = p.sw2 + (size_t)block_row * p.ldsw2;
    float next_g = __ldg(sg), next_u = __ldg(su);
    int from = 0;
#pragma unroll 1
    for (int n = 0; n < p.G; ++n) {
        const float s_g = next_g, s_u = next_u;
        if (n + 1 < p.G) { next_g = __ldg(sg + n + 1); next_u = __ldg(su + n + 1); }
        cp_async_wait<DEPTH - 2>();
        Chunk chunk;
        chunk.read(own + from * CHUNK);
        from = from + 1 == DEPTH ? 0 : from + 1;
        ask_w();
        ask_x();
        fp8_add_group<2, H>(chunk, total, sx + n * 8 * H + 2 * tq, s_g, s_u);
    }
    cp_async_wait<0>();
    float act[H][2];
    uint32_t m[H][2];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            act[h][e] = silu_f32<float>(total[0][h][e]) * total[0][h][2 + e];
            if (unit >= p.N) act[h][e] = 0.f;
            m[h][e] = fp8_magnitude(act[h][e]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) m[h][e] = max(m[h][e], __shfl_xor_sync(0xffffffffu, m[h][e], o));
        }
    cluster_wait();
    const int at = cluster_ctarank() * FG_WARPS + warp;
    if (g < 4) {        // (one row of lanes for each block of the cluster)
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                cluster_store_f32(cluster_map(smem_u32(&most[at][8 * h + 2 * tq + e]), g), __uint_as_float(m[h][e]));
    }
    cluster_sync_all();
    const int rank = cluster_ctarank();
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int j = 8 * h + 2 * tq + e, t = t0 + j;
            uint32_t a = 0;
#pragma unroll
            for (int i = 0; i < FG_WARPS * 4; ++i) a = max(a, most[i][j]);
            const Fp8Scale k = fp8_scale(a);
            codes[j][warp * 8 + g] = (uint8_t)fp8_pack4(act[h][e], 0.f, 0.f, 0.f, k.r);
            if (rank == 0 && warp == 0 && g == 0 && t < p.M) p.so[t * p.ldso + u0 / FP8_GROUP] = k.s;
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * H * FG_WARPS * 8; i += FG_WARPS * 32) {
        const int j = i / (FG_WARPS * 8), u = i - j * (FG_WARPS * 8);
        if (t0 + j < p.M && u0 + u < p.N) reinterpret_cast<uint8_t*>(p.out)[(t0 + j) * p.ldo + u0 + u] = codes[j][u];
    }
}

template <int R, int H, int DEPTH>
static int fr_launch(const Fp8RowsParams& p, int sms, cudaStream_t stream) {
    const int smem = RR_WARPS * DEPTH * RrChunk<R, H>::BYTES + p.G * 8 * H * 4;
    constexpr int fixed = 2 * RR_WARPS * 8 * H * (8 * R + 4) * 4 + 1024;
    if (smem + fixed > 227 * 1024) return ACV_ERR_SIZE;
    static AcvSmemConfig cfg;
    auto kernel = gemm_fp8_rows_kernel<R, H, DEPTH>;
    if (const int e = acv_ensure_smem(cfg, kernel, smem)) return e;
    const int resident = 228 * 1024 / (smem + fixed) >= 2 ? 2 : 1, tiles = (p.N + 8 * R - 1) / (8 * R);
    acv_launch(PDL_GEMM, kernel, dim3(min(tiles, resident * sms), (p.M + 8 * H - 1) / (8 * H)), dim3(RR_WARPS * 32), smem, stream, p);
    return acv_launch_status();
}
template <int H, int DEPTH>
static int fg_launch(const Fp8RowsParams& p, cudaStream_t stream) {
    const int smem = FG_WARPS * DEPTH * RrChunk<2, H>::BYTES + p.G * 8 * H * 4;
    if (smem > 200 * 1024) return ACV_ERR_SIZE;
    static AcvSmemConfig cfg;
    auto kernel = gemm_fp8_rows_gated_kernel<H, DEPTH>;
    if (const int e = acv_ensure_smem(cfg, kernel, smem)) return e;
    const int groups = (p.N + FP8_GROUP - 1) / FP8_GROUP;
    acv_launch_cluster(PDL_GEMM, dim3(4, 1, 1), kernel, dim3(groups * 4, (p.M + 8 * H - 1) / (8 * H)), dim3(FG_WARPS * 32), smem, stream, p);
    return acv_launch_status();
}

int acv_fp8_rows(const Fp8Operands& o, int flags, int sms, cudaStream_t stream) {
    Fp8RowsParams p = {};
    static_cast<Fp8Operands&>(p) = o;
    p.G = (p.K + FP8_GROUP - 1) / FP8_GROUP;
    p.early_w = flags & 1;
    if ((p.M + 7) / 8 > 65535) return ACV_ERR_SIZE;
    if (p.w2) return p.M > 8 ? fg_launch<2, 6>(p, stream) : fg_launch<1, 6>(p, stream);
    return p.M > 8 ? fr_launch<4, 2, 3>(p, sms, stream) : fr_launch<4, 1, 3>(p, sms, stream);
}
