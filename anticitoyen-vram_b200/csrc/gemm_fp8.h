// What the two files of 8-bit products share: a product's operands, and the streaming kernel's way in.
#pragma once

#include "common.cuh"

struct Fp8Operands {
    const uint8_t *x, *w, *w2;          // [M,K], [N,K]; w2: the up rows of the gated form
    const float *sx, *sw, *sw2;         // [M][G], [blocks of N][G]
    void* out;
    float* so;                          // gated: the scales of the quantised result
    long long ldx, ldw, ldw2, ldo, ldsx, ldsw, ldsw2, ldso;
    int M, N, K, out_f32;
};

int acv_fp8_rows(const Fp8Operands& o, int flags, cudaStream_t stream);
