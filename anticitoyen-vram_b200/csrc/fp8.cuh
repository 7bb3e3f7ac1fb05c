// e4m3 values with a float scale for each group of 128 (of a row) or block of 128 x 128 (of a weight).
//
//   a = max |x| over the group,  s = max(a / 448, 2^-126),  r = 1 / s,  q = e4m3(x r)        (448: the largest e4m3 number)
//
// Every step is a correctly rounded float operation, so q and s depend on the group's values alone.  The floor of 2^-126 keeps s
// a normal number, r finite and a group of zeros at q = 0.  A group that holds a NaN has s = NaN and every q NaN; one that holds an
// infinity has s = inf, its finite values become 0 and the infinity NaN: whatever product reads the row then gives NaN.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

#define FP8_GROUP 128

struct Fp8Scale { float s, r; };

// `amax`: the bits of the group's largest magnitude; magnitudes are ordered as their bits are, NaNs above infinity
__device__ __forceinline__ Fp8Scale fp8_scale(uint32_t amax) {
    float s = __fdiv_rn(__uint_as_float(amax), 448.f);
    if (s < 1.17549435e-38f) s = 1.17549435e-38f;
    return {s, __frcp_rn(s)};
}
__device__ __forceinline__ uint32_t fp8_magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// four values times r as e4m3, the first in the lowest byte (beyond 448 by the rounding of r alone: that is 448; NaN stays NaN)
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d, float r) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a * r, b * r), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c * r, d * r), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// ----------------------------------------------------------------------------- eight neighbouring elements of a row, float or bfloat16
// The bytes as they come from memory: converted where they are used, so that several loads are under way at once.
struct Raw8 { uint4 a, b; };
__device__ __forceinline__ Raw8 raw8_load(const void* row, int f32, int at) {
    Raw8 r;
    if (f32) {
        const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(row) + at);
        r.a = p[0];
        r.b = p[1];
    } else {
        r.a = *reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(row) + at);
        r.b = make_uint4(0, 0, 0, 0);
    }
    return r;
}
__device__ __forceinline__ void raw8_floats(const Raw8& r, int f32, float (&v)[8]) {
    const uint32_t a[4] = {r.a.x, r.a.y, r.a.z, r.a.w}, b[4] = {r.b.x, r.b.y, r.b.z, r.b.w};
    if (f32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = __uint_as_float(a[i]);
            v[4 + i] = __uint_as_float(b[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(a[i] << 16);
            v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
        }
    }
}
// Rows whose length, stride or start is not a multiple of 16 bytes go element by element.  The sixteen lanes of a group of 128 then take
// neighbouring elements, so that a load or store of a warp is two runs of sixteen: a lane's eight are 16 apart.
template <bool VEC>
__device__ __forceinline__ int piece_at(int piece) { return VEC ? piece * 8 : (piece & ~15) * 8 + (piece & 15); }
template <bool VEC>
__device__ __forceinline__ int piece_element(int at, int i) { return VEC ? at + i : at + 16 * i; }
// eight elements of a row in that order, zeros from `n` on
__device__ __forceinline__ void load8_ragged(const void* row, int f32, int at, int n, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i] = at + 16 * i >= n ? 0.f : f32 ? reinterpret_cast<const float*>(row)[at + 16 * i] : __bfloat162float(reinterpret_cast<const bf16*>(row)[at + 16 * i]);
}
__device__ __forceinline__ Raw8 raw8_load_ragged(const void* row, int f32, int at, int n) {
    uint32_t w[8] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (at + 16 * i < n) {
            if (f32) w[i] = reinterpret_cast<const uint32_t*>(row)[at + 16 * i];
            else w[i >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[at + 16 * i] << (16 * (i & 1));
        }
    return {make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7])};
}
__device__ __forceinline__ void store8(void* row, int f32, int at, const float (&v)[8]) {
    if (f32) {
        float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(row) + at);
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&b);
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<bf16*>(row) + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
__device__ __forceinline__ void store8_ragged(void* row, int f32, int at, int n, const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (at + 16 * i < n) {
            if (f32) reinterpret_cast<float*>(row)[at + 16 * i] = v[i];
            else reinterpret_cast<bf16*>(row)[at + 16 * i] = __float2bfloat16_rn(v[i]);
        }
}
template <bool VEC>
__device__ __forceinline__ void store_q8(uint8_t* row, int at, int n, const float (&v)[8], float r) {
    const uint32_t lo = fp8_pack4(v[0], v[1], v[2], v[3], r), hi = fp8_pack4(v[4], v[5], v[6], v[7], r);
    if (VEC) {
        *reinterpret_cast<uint2*>(row + at) = make_uint2(lo, hi);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (at + 16 * i < n) row[at + 16 * i] = (uint8_t)((i < 4 ? lo : hi) >> (8 * (i & 3)));
    }
}
__device__ __forceinline__ uint32_t magnitude8(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, fp8_magnitude(v[i]));
    return m;
}
// the same of eight elements as they came from memory: bfloat16 magnitudes are ordered as their bits are, two at a time
__device__ __forceinline__ uint32_t magnitude8(const Raw8& r, int f32) {
    const uint32_t a[4] = {r.a.x, r.a.y, r.a.z, r.a.w}, b[4] = {r.b.x, r.b.y, r.b.z, r.b.w};
    if (f32) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, max(a[i] & 0x7fffffffu, b[i] & 0x7fffffffu));
        return m;
    }
    const uint32_t m = __vmaxu2(__vmaxu2(a[0] & 0x7fff7fffu, a[1] & 0x7fff7fffu), __vmaxu2(a[2] & 0x7fff7fffu, a[3] & 0x7fff7fffu));
    return max(m << 16, m & 0xffff0000u);
}
// the largest over the sixteen lanes that hold a group of 128
__device__ __forceinline__ uint32_t half_warp_max(uint32_t m) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}
// g sigmoid(g) in front of a rounding to e4m3 whose scale it decides, exponential and quotient by the hardware's approximations: the
// exponential is off by 2 + 1.2 |g| units of a float, the quotient by two.  The first counts where g < 0: at g = -60 the value, and the scale
// of a group whose gates are all there, are off by 80 units (1e-5 of them; half a step of e4m3 is 6e-2), around 0 by five;
// in absolute numbers that is less than 3e-7 for every g < 0.  Beyond 2^126 in the denominator (g under -87.3) the quotient is 0, where the
// value is under 1e-36.  With the exact functions 2048 tokens of 12288 units take 268 us, not 250.
__device__ __forceinline__ float fp8_silu(float g) { return __fdividef(g, 1.f + __expf(-g)); }
static inline bool fp8_rows_aligned(const void* p, long long ld, int bytes, int to) {
    return !((uintptr_t)p % to) && !(ld * bytes % to);
}
