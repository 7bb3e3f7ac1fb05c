// Quantisation to e4m3: rows in groups of 128 (what a product's activations are) and blocks of 128 x 128 (its weights).
// The formulas stand in fp8.cuh.  Both forms read every element once and write a byte for it: memory bounds them.
#include "fp8.cuh"

// Rows: sixteen lanes hold a group, eight neighbouring elements each, so the group's maximum takes four exchanges and no shared
// memory.  A half-warp takes U groups at once, and asks for its next U before it works on them, so that loads are always under way; it goes
// on by the grid's stride, in (rows, groups) from the host, so no group costs a division for its place.  The scales' two divisions cost more
// than the rest of a group together: a half-warp's lanes make those of its U groups side by side, once.
// TYPE: of the elements, 0 bfloat16, 1 float, 2 as `said`.  4096 x 8192 bfloat16: 18.0 us, 5.6 TB/s; with two, four and six groups at once and as
// many blocks to an SM as their registers let be 20.2, 18.7, 18.8; four without the loads ahead 19.3.
template <bool VEC, int U, int TYPE>
__global__ void __launch_bounds__(256, 4) quantize_rows_kernel(const void* __restrict__ x, int said, long long ldx, uint8_t* __restrict__ q,
                                                               long long ldq, float* __restrict__ s, long long lds, int T, int K, int G,
                                                               int step_rows, int step_groups) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 15, f32 = TYPE == 2 ? said : TYPE;
    const size_t esz = f32 ? 4 : 2;
    const long long first = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
    int row = (int)(first / G), g = (int)(first - (long long)row * G);
    auto fetch = [&](int (&rows)[U], int (&gs)[U], Raw8 (&raw)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            rows[u] = row;
            gs[u] = g;
            row += step_rows;
            g += step_groups;
            if (g >= G) { g -= G; ++row; }
            const int at = piece_at<VEC>(gs[u] * 16 + lane);
            const char* src = reinterpret_cast<const char*>(x) + (size_t)rows[u] * ldx * esz;
            raw[u].a = raw[u].b = make_uint4(0, 0, 0, 0);
            if (rows[u] < T && at < K) {
                if (VEC) raw[u] = raw8_load(src, f32, at);
                else raw[u] = raw8_load_ragged(src, f32, at, K);
            }
        }
    };
    int rows[2][U], gs[2][U];
    Raw8 raw[2][U];
    auto finish = [&](int (&rows)[U], int (&gs)[U], Raw8 (&raw)[U]) {
        float v[8];
        uint32_t own = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t m = half_warp_max(magnitude8(raw[u], f32));
            if (lane % U == u) own = m;
        }
        const Fp8Scale mine = fp8_scale(own);           // of group lane % U
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float r = __shfl_sync(0xffffffffu, mine.r, u, 16);
            const int at = piece_at<VEC>(gs[u] * 16 + lane);
            if (rows[u] < T) {
                if (at < K) {
                    raw8_floats(raw[u], f32, v);
                    store_q8<VEC>(q + (size_t)rows[u] * ldq, at, K, v, r);
                }
                if (lane == u) s[(size_t)rows[u] * lds + gs[u]] = mine.s;
            }
        }
    };
    fetch(rows[0], gs[0], raw[0]);
    while (true) {
        if (!__any_sync(0xffffffffu, rows[0][0] < T)) break;
        fetch(rows[1], gs[1], raw[1]);
        finish(rows[0], gs[0], raw[0]);
        if (!__any_sync(0xffffffffu, rows[1][0] < T)) break;
        fetch(rows[0], gs[0], raw[0]);
        finish(rows[1], gs[1], raw[1]);
    }
}

// Blocks: 256 threads hold a block of 128 x 128 in registers (eight rows of eight elements a thread) between its maximum and its
// quantised values, so it is read once.  TYPE as above: half the registers in bfloat16, so more blocks to an SM.
template <bool VEC, int TYPE>
__global__ void __launch_bounds__(256) quantize_blocks_kernel(const void* __restrict__ x, int said, long long ldx, uint8_t* __restrict__ q,
                                                              long long ldq, float* __restrict__ s, long long lds, int T, int K) {
    __shared__ uint32_t red[8];
    pdl_launch_dependents();
    pdl_wait();
    const int at = piece_at<VEC>(blockIdx.x * 16 + (threadIdx.x & 15));
    const int row0 = blockIdx.y * FP8_GROUP + (threadIdx.x >> 4), f32 = TYPE == 2 ? said : TYPE;
    const size_t esz = f32 ? 4 : 2;
    Raw8 raw[8];
    float v[8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        raw[i].a = raw[i].b = make_uint4(0, 0, 0, 0);
        if (row0 + 16 * i < T && at < K) {
            const char* src = reinterpret_cast<const char*>(x) + (size_t)(row0 + 16 * i) * ldx * esz;
            raw[i] = VEC ? raw8_load(src, f32, at) : raw8_load_ragged(src, f32, at, K);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, magnitude8(raw[i], f32));
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, red[i]);
    const Fp8Scale k = fp8_scale(m);
    if (threadIdx.x == 0) s[(size_t)blockIdx.y * lds + blockIdx.x] = k.s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = row0 + 16 * i;
        if (row >= T || at >= K) continue;
        raw8_floats(raw[i], f32, v);
        store_q8<VEC>(q + (size_t)row * ldq, at, K, v, k.r);
    }
}

// x [T,K] float or bfloat16, rows dense at stride ldx; q [T,K] bytes at stride ldq; s: block_rows 1: [T][groups of K] at stride lds,
// 128: [blocks of T][groups of K].  (One record, field for field as kernels/ops.py packs it.)
struct QuantizeFp8Args {
    const void *x, *q, *s, *stream;
    long long ldx, ldq, lds;
    int dtype, T, K, block_rows, sms;
};
ACV_API int acv_quantize_fp8(const QuantizeFp8Args* a) {
    const void* x = a->x;
    uint8_t* q = (uint8_t*)const_cast<void*>(a->q);
    float* s = (float*)const_cast<void*>(a->s);
    const long long ldx = a->ldx, ldq = a->ldq, lds = a->lds;
    const int dtype = a->dtype, T = a->T, K = a->K, block_rows = a->block_rows, sms = a->sms;
    const cudaStream_t stream = (cudaStream_t)const_cast<void*>(a->stream);
    if (T <= 0 || K <= 0) return 0;
    if (K > 0x7fffffff - 1024) return ACV_ERR_SIZE;         // (rounded up to groups in 32 bits)
    if (dtype != ACV_F32 && dtype != ACV_BF16) return ACV_ERR_DTYPE;
    const int f32 = dtype == ACV_F32;
    const int G = (K + FP8_GROUP - 1) / FP8_GROUP;
    const bool vec = K % 8 == 0 && fp8_rows_aligned(x, ldx, f32 ? 4 : 2, 16) && fp8_rows_aligned(q, ldq, 1, 8);
    if (block_rows == FP8_GROUP) {
        const long long down = ((long long)T + FP8_GROUP - 1) / FP8_GROUP;
        if (down > 65535) return ACV_ERR_SIZE;
        const dim3 grid(G, (unsigned)down);
        if (!vec) acv_launch(PDL_MISC, quantize_blocks_kernel<false, 2>, grid, 256, 0, stream, x, f32, ldx, q, ldq, s, lds, T, K);
        else if (f32) acv_launch(PDL_MISC, quantize_blocks_kernel<true, 1>, grid, 256, 0, stream, x, f32, ldx, q, ldq, s, lds, T, K);
        else acv_launch(PDL_MISC, quantize_blocks_kernel<true, 0>, grid, 256, 0, stream, x, f32, ldx, q, ldq, s, lds, T, K);
        return acv_launch_status();
    }
    if (block_rows != 1) return ACV_ERR_SIZE;
    const long long groups = (long long)T * G;
    const long long blocks = (groups + 15) / 16;
    const int grid = (int)(blocks < (long long)sms * 4 ? blocks : (long long)sms * 4);
    const long long stride = (long long)grid * 16;
    const int step_rows = (int)(stride / G), step_groups = (int)(stride % G);
    if ((long long)T + 8ll * (step_rows + 1) > 0x7fffffffll) return ACV_ERR_SIZE;
    if (!vec)
        acv_launch(PDL_MISC, quantize_rows_kernel<false, 2, 2>, grid, 256, 0, stream, x, f32, ldx, q, ldq, s, lds, T, K, G, step_rows, step_groups);
    else if (f32)
        acv_launch(PDL_MISC, quantize_rows_kernel<true, 2, 1>, grid, 256, 0, stream, x, f32, ldx, q, ldq, s, lds, T, K, G, step_rows, step_groups);
    else
        acv_launch(PDL_MISC, quantize_rows_kernel<true, 3, 0>, grid, 256, 0, stream, x, f32, ldx, q, ldq, s, lds, T, K, G, step_rows, step_groups);
    return acv_launch_status();
}
