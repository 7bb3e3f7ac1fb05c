// The products of e4m3 operands with block scales for up to sixteen tokens and weights of one round of blocks: every weight is read
// once, and what bounds them beside that is what comes before the first and after the last of them.
//
//   y[t][n] = sum over groups g of 128 k of  sx[t][g] sw[n / 128][g] sum over k in g of qx[t][k] qw[n][k]
//
// A block takes 32 weight rows and its eight warps an eighth of the groups each.  A group's inner sum is four mma.sync of 32 k (weight
// rows are its M, tokens its N) into float; the two scales multiply it as it joins the running float sum.  As in gemm_rows.cu a lane
// brings its own operands by 16-byte asynchronous copies into a ring that it alone reads, so no barrier stands in the loop: a group of a
// row is 128 bytes, as 64 bfloat16 are, and the ring's layout is the same.  Which k of a group a lane holds is the same for tokens and
// weights.  The tokens' scales of a warp's groups are fetched once, into shared memory of its own.
//
// Beside tiles of 128 weight rows on tcgen05 (gemm_fp8_narrow.cu), microseconds here and there, 8 tokens: 1024 x 1024 2.1 and 3.1,
// 4096 x 2560 3.4 and 4.5, 4096 x 4096 4.2 and 5.4, 4096 x 12288 11.6 and 11.2; with a second round of blocks (6144 x 4096) 7.6 and 5.8.
// An mma.sync of this type takes its operands apart into several instructions: that is what a block's time goes to.
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
__device__ __forceinline__ void fp8_add_group(const RrChunk<R, H>& k, float (&total)[R / 2][H][4], const float* sx, float sw) {
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
            const float s0 = sx[8 * h] * sw, s1 = sx[8 * h + 1] * sw;
            total[a][h][0] = fmaf(c[0], s0, total[a][h][0]);
            total[a][h][1] = fmaf(c[1], s1, total[a][h][1]);
            total[a][h][2] = fmaf(c[2], s0, total[a][h][2]);
            total[a][h][3] = fmaf(c[3], s1, total[a][h][3]);
        }
}

// H: octets of tokens; DEPTH: groups in a warp's ring
#define FR_ROWS 4           // octets of weight rows of a block
template <int H, int DEPTH>
__global__ void __launch_bounds__(RR_WARPS * 32, 2) gemm_fp8_rows_kernel(const Fp8RowsParams p) {
    using Chunk = RrChunk<FR_ROWS, H>;
    constexpr int CHUNK = Chunk::BYTES, COLS = 8 * FR_ROWS;
    extern __shared__ __align__(16) unsigned char ring[];
    __shared__ float part[1][RR_WARPS][8 * H][COLS + 4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
    const int n0 = blockIdx.x * COLS;
    const int c0 = p.G * warp / RR_WARPS, chunks = p.G * (warp + 1) / RR_WARPS - c0;
    const uint32_t own = smem_u32(ring) + warp * (DEPTH * CHUNK) + lane * 16;
    float* sx = reinterpret_cast<float*>(ring + RR_WARPS * DEPTH * CHUNK) + (size_t)c0 * 8 * H;      // [its groups][8 H tokens]
    int w_next = 0, w_into = 0, x_next = 0, x_into = 0;
    auto ask_w = [&]() {
        if (w_next >= chunks) return;
        const uint32_t dst = own + w_into * CHUNK;
        const int k = (c0 + w_next) * FP8_GROUP + tq * 16;
#pragma unroll
        for (int r = 0; r < FR_ROWS; ++r) {
            const int row = n0 + r * 8 + g;
            const uint8_t* src = p.w + (size_t)min(row, p.N - 1) * p.ldw;
#pragma unroll
            for (int b = 0; b < 2; ++b) copy16_of_row(Chunk::weights_at(dst, b, r), src, k + b * 64, p.K, row < p.N);
        }
        w_into = w_into + 1 == DEPTH ? 0 : w_into + 1;
        ++w_next;
    };
    auto ask_x = [&]() {
        if (x_next < chunks) {
            const uint32_t dst = own + x_into * CHUNK;
            const int k = (c0 + x_next) * FP8_GROUP + tq * 16;
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const int t = h * 8 + g;
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
    pdl_launch_dependents();
    pdl_wait();
#pragma unroll
    for (int i = 0; i < DEPTH - 1; ++i) {
        if (!p.early_w) ask_w();
        ask_x();
    }
    for (int i = lane; i < chunks * 8 * H; i += 32) {
        const int t = i % (8 * H);
        sx[i] = t < p.M ? p.sx[t * p.ldsx + c0 + i / (8 * H)] : 0.f;
    }
    __syncwarp();
    float total[FR_ROWS / 2][H][4];
#pragma unroll
    for (int a = 0; a < FR_ROWS / 2; ++a)
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) total[a][h][i] = 0.f;
    const float* sw = p.sw + (size_t)(n0 / FP8_GROUP) * p.ldsw + c0;
    float scale = chunks ? sw[0] : 0.f;
    int from = 0;
#pragma unroll 1
    for (int n = 0; n < chunks; ++n) {
        const float s = scale;
        if (n + 1 < chunks) scale = sw[n + 1];
        cp_async_wait<DEPTH - 2>();
        Chunk chunk;
        chunk.read(own + from * CHUNK);
        from = from + 1 == DEPTH ? 0 : from + 1;
        ask_w();
        ask_x();
        fp8_add_group<FR_ROWS, H>(chunk, total, sx + n * 8 * H + 2 * tq, s);
    }
    cp_async_wait<0>();
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int r = 0; r < FR_ROWS; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) part[0][warp][h * 8 + 2 * tq + e][r * 8 + g] = total[r / 2][h][2 * (r & 1) + e];
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * H * COLS; i += RR_WARPS * 32) {
        const int t = i / COLS, q = i - t * COLS, n = n0 + q;
        if (t >= p.M || n >= p.N) continue;
        const float v = rr_sum(part[0], t, q);
        if (p.out_f32) reinterpret_cast<float*>(p.out)[t * p.ldo + n] = v;
        else reinterpret_cast<bf16*>(p.out)[t * p.ldo + n] = __float2bfloat16_rn(v);
    }
}

template <int H, int DEPTH>
static int fr_launch(const Fp8RowsParams& p, cudaStream_t stream) {
    constexpr int COLS = 8 * FR_ROWS;
    const int smem = RR_WARPS * DEPTH * RrChunk<FR_ROWS, H>::BYTES + p.G * 8 * H * 4;
    if (smem + RR_WARPS * 8 * H * (COLS + 4) * 4 + 1024 > 227 * 1024) return ACV_ERR_SIZE;
    static AcvSmemConfig cfg;
    auto kernel = gemm_fp8_rows_kernel<H, DEPTH>;
    if (const int e = acv_ensure_smem(cfg, kernel, smem)) return e;
    acv_launch(PDL_GEMM, kernel, dim3((p.N + COLS - 1) / COLS), dim3(RR_WARPS * 32), smem, stream, p);
    return acv_launch_status();
}

int acv_fp8_rows(const Fp8Operands& o, int flags, cudaStream_t stream) {
    if (o.w2 || o.M > 16) return ACV_ERR_SIZE;
    Fp8RowsParams p = {};
    static_cast<Fp8Operands&>(p) = o;
    p.G = (p.K + FP8_GROUP - 1) / FP8_GROUP;
    p.early_w = flags & 1;
    return p.M > 8 ? fr_launch<2, 3>(p, stream) : fr_launch<1, 3>(p, stream);
}
