// The step between two parts of a layer: what the part before leaves joins the stream, and the part behind gets its norm.
//
//   n = d / sqrt(mean(d^2) + e1) * w1         (the norm behind the part; without w1 n = d)
//   x += c * (g * n)                          (c: one number, g: a number for each channel or for each channel of each token)
//   h = x / sqrt(mean(x^2) + e2) * w2         (the norm in front of the next part, of the stream as it is kept; optional)
//
// h is rounded once, to float, bfloat16, or e4m3 with a scale for each group of 128 (fp8.cuh), which is what an 8-bit product reads.
// One block a row; a thread keeps its elements (eight neighbouring ones, C such pieces) in registers from their only read to their
// only write, both statistics are 32-bit sums over the block.  Sixteen neighbouring lanes hold a group, so its maximum takes four
// exchanges.  Memory bounds it with many rows, the chain load - sum - sum - store with few.
#include "fp8.cuh"

struct GnParams {
    void* x;
    const void *d, *g;
    const float *w1, *w2, *gc;
    void* out;
    float* s;
    long long ldx, ldd, ldg, ldo, lds;
    int H, x_f32, d_f32, g_f32, out_kind;       // out_kind: 0 float, 1 bfloat16, 2 e4m3, 3 none
    int early_w;                                // the weights may be read before the kernel in front has ended
    float c, e1, e2, inv_h;
};

// XT, DT: the stream's and the part's element type, 0 bfloat16, 1 float, 2 as the parameters say (a type known when the kernel is built
// halves what a row costs in instructions, which is what bounds many rows beside memory)
template <int TYPE>
__device__ __forceinline__ int gn_f32(int said) { return TYPE == 2 ? said : TYPE; }
template <bool VEC>
__device__ __forceinline__ void gn_load(const void* row, int f32, int at, int H, float (&v)[8]) {
    if (VEC) raw8_floats(raw8_load(row, f32, at), f32, v);
    else load8_ragged(row, f32, at, H, v);
}

// A row whose pieces are in `xw`, `dw` and `gw` (VEC), or are read here element by element.  C: pieces of eight elements a thread; with
// one the weights are in `w1`, `w2` and `gc` already, with more they are read where they are used.
template <bool VEC, int C, int XT, int DT>
__device__ __forceinline__ void gn_row(const GnParams& p, size_t row, const Raw8 (&xw)[C], const Raw8 (&dw)[C], const Raw8 (&gw)[C],
                                       float (&w1)[8], float (&w2)[8], float (&gc)[8], float* red) {
    const int H = p.H, x_f32 = gn_f32<XT>(p.x_f32), d_f32 = gn_f32<DT>(p.d_f32);
    char* xr = reinterpret_cast<char*>(p.x) + row * p.ldx * (x_f32 ? 4 : 2);
    const char* dr = reinterpret_cast<const char*>(p.d) + row * p.ldd * (d_f32 ? 4 : 2);
    const char* gr = p.g ? reinterpret_cast<const char*>(p.g) + row * p.ldg * (p.g_f32 ? 4 : 2) : nullptr;
    float x[C][8], d[C][8];
    if (p.d) {
        float r = 1.f;
        if (p.w1) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const int at = piece_at<VEC>(threadIdx.x + i * blockDim.x);
                if (at < H) {
                    if (VEC) raw8_floats(dw[i], d_f32, d[i]);
                    else load8_ragged(dr, d_f32, at, H, d[i]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) ss = fmaf(d[i][e], d[i][e], ss);
                }
            }
            ss = block_sum(ss, red);
            r = rsqrtf(fmaf(ss, p.inv_h, p.e1));
        }
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int at = piece_at<VEC>(threadIdx.x + i * blockDim.x);
            if (at >= H) continue;
            if (p.w1) {
                if (C > 1) gn_load<VEC>(p.w1, 1, at, H, w1);
#pragma unroll
                for (int e = 0; e < 8; ++e) d[i][e] = d[i][e] * r * w1[e];
            } else {
                if (VEC) raw8_floats(dw[i], d_f32, d[i]);
                else load8_ragged(dr, d_f32, at, H, d[i]);
            }
            if (gr) {
                float g[8];
                if (!VEC) load8_ragged(gr, p.g_f32, at, H, g);
                else if (p.g_f32) raw8_floats(gw[i], 1, g);
                else raw8_floats(gw[i], 0, g);
#pragma unroll
                for (int e = 0; e < 8; ++e) d[i][e] *= g[e];
            } else if (p.gc) {
                if (C > 1) gn_load<VEC>(p.gc, 1, at, H, gc);
#pragma unroll
                for (int e = 0; e < 8; ++e) d[i][e] *= gc[e];
            }
            if (VEC) raw8_floats(xw[i], x_f32, x[i]);
            else load8_ragged(xr, x_f32, at, H, x[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[i][e] = fmaf(p.c, d[i][e], x[i][e]);
                if (!x_f32) x[i][e] = round_to<bf16>(x[i][e]);
            }
            if (VEC) store8(xr, x_f32, at, x[i]);
            else store8_ragged(xr, x_f32, at, H, x[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int at = piece_at<VEC>(threadIdx.x + i * blockDim.x);
            if (at >= H) continue;
            if (VEC) raw8_floats(xw[i], x_f32, x[i]);
            else load8_ragged(xr, x_f32, at, H, x[i]);
        }
    }
    if (p.out_kind == 3) return;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i)
        if (piece_at<VEC>(threadIdx.x + i * blockDim.x) < H) {
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(x[i][e], x[i][e], ss);
        }
    ss = block_sum(ss, red);
    const float r = rsqrtf(fmaf(ss, p.inv_h, p.e2));
    char* o = reinterpret_cast<char*>(p.out) + row * p.ldo * (p.out_kind == 0 ? 4 : p.out_kind == 1 ? 2 : 1);
    uint32_t own = 0;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int at = piece_at<VEC>(threadIdx.x + i * blockDim.x);
        const bool in = at < H;
        if (C > 1 && in) gn_load<VEC>(p.w2, 1, at, H, w2);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = (VEC ? in : piece_element<VEC>(at, e) < H) ? x[i][e] * r * w2[e] : 0.f;      // (zeros behind the row's end)
        if (p.out_kind == 2) {          // (whole warps pass here)
            const uint32_t m = half_warp_max(magnitude8(x[i]));
            if ((int)(threadIdx.x % C) == i) own = m;
        } else if (in) {
            if (VEC) store8(o, p.out_kind == 0, at, x[i]);
            else store8_ragged(o, p.out_kind == 0, at, H, x[i]);
        }
    }
    if (p.out_kind != 2) return;
    // the scales of a half-warp's C groups, made side by side by its lanes
    const Fp8Scale mine = fp8_scale(own);
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int at = piece_at<VEC>(threadIdx.x + i * blockDim.x);
        const float k = __shfl_sync(0xffffffffu, mine.r, i, 16);
        if (at < H) store_q8<VEC>(reinterpret_cast<uint8_t*>(o), at, H, x[i], k);
        const int group = (int)((threadIdx.x & ~15u) + i * blockDim.x) / 16;
        if ((int)(threadIdx.x & 15) == i && group * FP8_GROUP < H) p.s[row * p.lds + group] = mine.s;
    }
}

// A block a row.  BLOCKS of 512 threads have to fit an SM: 2 holds a thread to 64 registers.
template <bool VEC, int C, int XT, int DT, int BLOCKS>
__global__ void __launch_bounds__(512, BLOCKS) gated_norms_kernel(const GnParams p) {
    __shared__ float red[32];
    pdl_launch_dependents();
    const int H = p.H;
    float w1[8], w2[8], gc[8];
    auto weights = [&]() {
        const int at = piece_at<VEC>(threadIdx.x);
        if (C > 1 || at >= H) return;
        if (p.w1) gn_load<VEC>(p.w1, 1, at, H, w1);
        if (p.w2) gn_load<VEC>(p.w2, 1, at, H, w2);
        if (p.gc) gn_load<VEC>(p.gc, 1, at, H, gc);
    };
    if (p.early_w) weights();
    pdl_wait();
    const size_t row = blockIdx.x;
    Raw8 xw[C], dw[C], gw[C];
    if (VEC) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int at = piece_at<VEC>(threadIdx.x + i * blockDim.x);
            if (at < H) {
                const int x_f32 = gn_f32<XT>(p.x_f32), d_f32 = gn_f32<DT>(p.d_f32);
                if (p.d) dw[i] = raw8_load(reinterpret_cast<const char*>(p.d) + row * p.ldd * (d_f32 ? 4 : 2), d_f32, at);
                xw[i] = raw8_load(reinterpret_cast<const char*>(p.x) + row * p.ldx * (x_f32 ? 4 : 2), x_f32, at);
                if (p.g) gw[i] = raw8_load(reinterpret_cast<const char*>(p.g) + row * p.ldg * (p.g_f32 ? 4 : 2), p.g_f32, at);
            }
        }
    }
    if (!p.early_w) weights();
    gn_row<VEC, C, XT, DT>(p, row, xw, dw, gw, w1, w2, gc, red);
}

// Pieces of eight elements a thread: with few rows one as long as 512 threads cover a row, for a row's time is then its chain of loads,
// sums and stores, and more warps bring it in sooner (150 rows of 5120 with one, two and two pieces at 64 registers: -, 4.8, 5.6 us; 300 of
// 4096: 3.7, 3.9, 3.9).  With many rows two, and as many blocks to an SM as 64 registers allow: what a warp does once for a row (sums over
// the block, the scales' divisions) serves more of it, and what is left of a row's time are its instructions (4096 rows of 4096, bfloat16 in,
// e4m3 out, with one, two and four pieces 34, 26, 32 us; of 5120, a float stream and a gate for every token 55, 49, 53, of which 45 is memory's).
template <bool VEC, int XT, int DT>
static int gn_launch(const GnParams& p, int T, int sms, cudaStream_t stream) {
    const int pieces = (p.H + 7) / 8;
    auto threads = [&](int c) { return ((pieces + c - 1) / c + 31) / 32 * 32; };
    const bool few = T <= 2 * sms;
    if (few && threads(1) <= 512) acv_launch(PDL_NORM, gated_norms_kernel<VEC, 1, XT, DT, 1>, T, threads(1), 0, stream, p);
    else if (few && threads(2) <= 512) acv_launch(PDL_NORM, gated_norms_kernel<VEC, 2, XT, DT, 1>, T, threads(2), 0, stream, p);
    else if (threads(2) <= 512) acv_launch(PDL_NORM, gated_norms_kernel<VEC, 2, XT, DT, 2>, T, threads(2), 0, stream, p);
    else if (threads(4) <= 512) acv_launch(PDL_NORM, gated_norms_kernel<VEC, 4, XT, DT, 1>, T, threads(4), 0, stream, p);
    else return ACV_ERR_SIZE;
    return acv_launch_status();
}

// x [T,H] in place; d [T,H] or null; gate: g [T,H] or gc float [H] or neither; w1 or null; out [T,H] of out_kind (0 float, 1 bfloat16,
// 2 e4m3 with scales s [T][groups of H], 3 none); every matrix's rows dense at a stride of its own.  (One record, field for field as
// kernels/ops.py packs it.)
struct GatedNormsArgs {
    const void *x, *d, *g, *gc, *w1, *w2, *out, *s, *stream;
    long long ldx, ldd, ldg, ldo, lds;
    int x_dtype, d_dtype, g_dtype, out_kind, T, H, sms, early_w;
    float c, e1, e2;
};
ACV_API int acv_add_gated_norms(const GatedNormsArgs* a) {
    const int T = a->T, H = a->H;
    if (T <= 0 || H <= 0) return 0;
    if ((a->x_dtype | a->d_dtype | a->g_dtype) & ~1) return ACV_ERR_DTYPE;
    if ((unsigned)a->out_kind > 3u || (a->out_kind < 3 && (!a->out || !a->w2)) || (a->out_kind == 2 && !a->s)) return ACV_ERR_DTYPE;
    GnParams p = {};
    p.x = const_cast<void*>(a->x); p.d = a->d; p.g = a->g; p.gc = a->g ? nullptr : (const float*)a->gc;
    p.w1 = a->d ? (const float*)a->w1 : nullptr; p.w2 = a->out_kind < 3 ? (const float*)a->w2 : nullptr;
    p.out = const_cast<void*>(a->out); p.s = (float*)const_cast<void*>(a->s);
    p.ldx = a->ldx; p.ldd = a->ldd; p.ldg = a->ldg; p.ldo = a->ldo; p.lds = a->lds; p.H = H;
    p.x_f32 = a->x_dtype == ACV_F32; p.d_f32 = a->d_dtype == ACV_F32; p.g_f32 = a->g_dtype == ACV_F32; p.out_kind = a->out_kind; p.early_w = a->early_w;
    p.c = a->c; p.e1 = a->e1; p.e2 = a->e2; p.inv_h = 1.f / (float)H;
    const int ob = p.out_kind == 0 ? 4 : p.out_kind == 1 ? 2 : 1;
    const bool vec = H % 8 == 0 && fp8_rows_aligned(p.x, p.ldx, p.x_f32 ? 4 : 2, 16) && (!p.d || fp8_rows_aligned(p.d, p.ldd, p.d_f32 ? 4 : 2, 16)) &&
                     (!p.g || fp8_rows_aligned(p.g, p.ldg, p.g_f32 ? 4 : 2, 16)) &&
                     (p.out_kind == 3 || fp8_rows_aligned(p.out, p.ldo, ob, p.out_kind == 2 ? 8 : 16)) &&
                     !(((uintptr_t)p.gc | (uintptr_t)p.w1 | (uintptr_t)p.w2) & 15);
    const cudaStream_t stream = (cudaStream_t)const_cast<void*>(a->stream);
    if (!vec) return gn_launch<false, 2, 2>(p, T, a->sms, stream);
    if (p.x_f32) return p.d_f32 ? gn_launch<true, 1, 1>(p, T, a->sms, stream) : gn_launch<true, 1, 0>(p, T, a->sms, stream);
    return p.d_f32 ? gn_launch<true, 0, 1>(p, T, a->sms, stream) : gn_launch<true, 0, 0>(p, T, a->sms, stream);
}
