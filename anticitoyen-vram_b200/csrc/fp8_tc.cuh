// What the tcgen05 kernels of 8-bit products share: their parameters, the issuing warp's and the epilogue's building blocks.
#pragma once

#include "fp8.cuh"
#include "gemm_fp8.h"
#include "tc_ptx.cuh"
#include "tensor_map.h"

#define FT_ROWS 128                         // rows of an operand tile = bytes of a k-block's row
#define FT_TILE (FT_ROWS * FT_ROWS)         // bytes of an operand tile of 128 rows

struct Fp8TcParams {
    int M, N, n_kb;                         // N: features, or units of the gated form
    const float *sx, *sw, *sw2;             // sw2: the up rows' scales of the gated form
    long long ldsx, ldsw, ldsw2, ldo, ldso;
    void* out;
    float* so;
    int out_f32, out_vec, sx_vec;           // _vec: rows of out take 16-byte stores, those of sx 16-byte loads
    int tiles_m, tiles_n, group, stages, splits, kb_per_split, early_w;
    int* status;
    unsigned int wait_limit;                // of polls; less and a k-block whose loads are left out (skip_kb >= 0) in the test of the waits only
    int skip_kb;
};

__device__ __forceinline__ uint32_t ft_idesc(int n, int m) {        // float accumulator, e4m3 operands (type 0), both K-major
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// One lane of a converged warp.  The issuing warp runs its loop as a whole and lets this lane issue: what the products need is then
// known to be the warp's and is kept in uniform registers.  (A loop run by one lane alone moved every descriptor there first: 600
// cycles a k-block, where the tensor core needs 512 for the largest.)
__device__ __forceinline__ bool ft_elect() {
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}
// a number in 0 .. 2^16 - 1 for each tile, neighbours far apart whatever it is divided by (Fibonacci hashing)
__device__ __forceinline__ unsigned int ft_spread(int tile) { return (unsigned int)tile * 0x9E3779B1u >> 16; }
__device__ __forceinline__ int ft_warp() { return __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0); }
template <bool PAIR>
__device__ __forceinline__ void ft_mma(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    if (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate) : "memory");
}
// the registers of a load are what its wait hands over: nothing that reads them moves in front of it
__device__ __forceinline__ void ft_wait_ld(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                   "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
__device__ __forceinline__ void ft_fma2(uint64_t& sum, uint32_t lo, uint32_t hi, uint64_t scale) {
    asm("{\n\t.reg .b64 v;\n\tmov.b64 v, {%1, %2};\n\tfma.rn.f32x2 %0, v, %3, %0;\n\t}" : "+l"(sum) : "r"(lo), "r"(hi), "l"(scale));
}
__device__ __forceinline__ uint64_t ft_both(float v) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "r"(__float_as_uint(v)));
    return r;
}
__device__ __forceinline__ uint64_t ft_pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(__float_as_uint(lo)), "r"(__float_as_uint(hi)));
    return r;
}
__device__ __forceinline__ float2 ft_floats(uint64_t v) {
    uint32_t lo, hi;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
    return make_float2(__uint_as_float(lo), __uint_as_float(hi));
}

// After a wait that ran out, by one warp, when every role has left its loop (before that nobody knows whether another will give up): what
// is still under way, loads that write into shared memory and products that read it, is waited for before the CTA's memory goes back,
// each stage by the parity of the last of the `uses` k-blocks that went into it.  `bars`: the stages' "full" barriers, uses: the k-blocks
// asked for; or the "empty" ones and the k-blocks whose products were issued.  The limit is this wait's own: a load is microseconds
// away however few polls the others were given, and one that never comes is not waited for longer than some 20 milliseconds (5 us a poll).
#define FT_DRAIN_LIMIT (1u << 12)
__device__ __forceinline__ void ft_drain(uint32_t bars, int stages, int uses) {
    for (int s = 0; s < stages && s < uses; ++s) {
        const int last = (uses - 1 - s) / stages;
        for (unsigned int i = 0; i < FT_DRAIN_LIMIT; ++i)
            if (mbar_try_wait(bars + 8 * s, last & 1)) break;
    }
}

// whether a phase is over, asked without waiting: the answer is a shared-memory access away, so it is asked for a turn ahead of its use
__device__ __forceinline__ bool ft_ready(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.b32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// a wait by a whole warp: true for all of its lanes where it ran out for one
__device__ __forceinline__ bool ft_warp_failed(uint32_t bar, uint32_t parity, volatile int* abort_flag, const Fp8TcParams& p, int code = 4) {
    const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, p.wait_limit));
    if (!ok && (threadIdx.x & 31) == 0) {
        *abort_flag = 1;
        atomicExch(p.status, code);
    }
    return !ok;
}

__device__ __forceinline__ float4 ft_read4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
// a number into another CTA's shared memory (there when the cluster has met)
__device__ __forceinline__ void ft_tell(uint32_t addr, int v) {
    asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ float4 ft_cluster_read4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// A tile's way out.  Every CTA of a cluster holds its share of the sums in its shared memory, float [token][BN features] with rows `ld`
// floats apart, at the same address `at`; they are added in rank order.  A warp takes the tokens first, first + step, ... < rows (the
// cluster's CTAs and their warps share them), a lane four neighbouring features.  GATED: the features are units' gates, then the same
// units' ups; a token's 128 units are a group and the warp holds it.  HALVES 1: a CTA has them all (BN 256); 2: it has 64 of them (BN 128),
// the CTAs of even rank the first 64, those of odd rank the others.
// AT_ONCE: tokens that a warp takes together (another CTA's shared memory is half a microsecond away under load; of the gated form's
// scales its lanes make one each, side by side).  SPLITS: the most shares a sum may have here; 1: the CTA is its whole cluster.
template <int BN, bool GATED, int HALVES, int AT_ONCE, int SPLITS>
__device__ __forceinline__ void ft_emit(const Fp8TcParams& p, uint32_t at, int ld, int first, int step, int rows, int row0, int tb) {
    const int lane = threadIdx.x & 31, half = HALVES == 2 ? lane >> 4 : 0;
    // the sums of features c .. c + 3 and the tokens r, r + step, ..
    auto sum4 = [&](int r, int c, float4 (&v)[AT_ONCE]) {
        if constexpr (SPLITS == 1 && HALVES == 1) {
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) v[j] = ft_read4(at + (uint32_t)(min(r + j * step, rows - 1) * ld + c) * 4);
        } else {
            float4 o[AT_ONCE][SPLITS];
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j)
#pragma unroll
                for (int q = 0; q < SPLITS; ++q)
                    if (q < p.splits)
                        o[j][q] = ft_cluster_read4(cluster_map(at + (uint32_t)(min(r + j * step, rows - 1) * ld + c) * 4, q * HALVES + half));
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                v[j] = o[j][0];
#pragma unroll
                for (int q = 1; q < SPLITS; ++q)
                    if (q < p.splits) { v[j].x += o[j][q].x; v[j].y += o[j][q].y; v[j].z += o[j][q].z; v[j].w += o[j][q].w; }
            }
        }
    };
#pragma unroll 1
    for (int r = first; r < rows; r += AT_ONCE * step) {
        if (GATED) {
            const int c = HALVES == 2 ? 4 * (lane & 15) : 4 * lane;
            float4 gs[AT_ONCE], us[AT_ONCE];
            sum4(r, c, gs);
            sum4(r, BN / 2 + c, us);
            uint32_t own = 0;
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                float4 &h = gs[j], &u = us[j];
                h.x = fp8_silu(h.x) * u.x; h.y = fp8_silu(h.y) * u.y; h.z = fp8_silu(h.z) * u.z; h.w = fp8_silu(h.w) * u.w;
                uint32_t m = max(max(fp8_magnitude(h.x), fp8_magnitude(h.y)), max(fp8_magnitude(h.z), fp8_magnitude(h.w)));
                m = __reduce_max_sync(0xffffffffu, m);
                if (lane % AT_ONCE == j) own = m;
            }
            const Fp8Scale k = fp8_scale(own);              // of token lane % AT_ONCE
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                const float by = __shfl_sync(0xffffffffu, k.r, j);
                if (r + j * step >= rows) break;
                const size_t row = (size_t)(row0 + r + j * step);
                const uint32_t w = fp8_pack4(gs[j].x, gs[j].y, gs[j].z, gs[j].w, by);
                if (lane == j) p.so[row * p.ldso + tb] = k.s;
                const int u0 = tb * FT_ROWS + 4 * lane;
                uint8_t* o = reinterpret_cast<uint8_t*>(p.out) + row * p.ldo + u0;
                if (p.out_vec && u0 + 4 <= p.N) {
                    *reinterpret_cast<uint32_t*>(o) = w;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (u0 + i < p.N) o[i] = (uint8_t)(w >> (8 * i));
                }
            }
        } else {
#pragma unroll
            for (int c = 4 * lane; c < BN; c += 128) {
                float4 vs[AT_ONCE];
                sum4(r, c, vs);
                const int n = tb * BN + c;
                if (n >= p.N) continue;
#pragma unroll
                for (int j = 0; j < AT_ONCE; ++j) {
                    if (r + j * step >= rows) break;
                    const size_t row = (size_t)(row0 + r + j * step);
                    const float4 v = vs[j];
                    const float f[4] = {v.x, v.y, v.z, v.w};
                    if (p.out_f32) {
                        float* o = reinterpret_cast<float*>(p.out) + row * p.ldo + n;
                        if (p.out_vec && n + 4 <= p.N) {
                            *reinterpret_cast<float4*>(o) = v;
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (n + i < p.N) o[i] = f[i];
                        }
                    } else {
                        bf16* o = reinterpret_cast<bf16*>(p.out) + row * p.ldo + n;
                        if (p.out_vec && n + 4 <= p.N) {
                            *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (n + i < p.N) o[i] = __float2bfloat16_rn(f[i]);
                        }
                    }
                }
            }
        }
    }
}

// tensor map of a matrix of bytes [rows, K] with row stride ld: box = 128 x box_rows, 128-byte swizzle
static inline int ft_map(CUtensorMap* map, const void* base, int rows, int K, long long ld, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return ACV_ERR_SIZE;
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {FT_ROWS, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : ACV_ERR_ALIGN;
}


// gemm_fp8_narrow.cu: tokens on the columns, `bt` of them (16 or 32) to a tile, K over `splits` CTAs
int acv_fp8_narrow(const CUtensorMap& mx, const CUtensorMap& mw, const CUtensorMap& mw2, Fp8TcParams& p, bool gated, int bt, int splits,
                   int sms, cudaStream_t stream);
