// What the kernels of the 8-bit floating-point product share (linear_f8.cu: few rows; linear_f8_tc.cu: many).
#pragma once

#include "f8.cuh"

namespace sxb {

struct F8Args {
    const uint8_t *x, *w;
    const float *xs, *ws;
    void *y;
    int64_t x_ld, xs_ld, y_ld, K;
    int M, N, kb;  // kb: blocks of 128 along k
    int f32;       // y is FP32, else BF16
};

// The form on tcgen05 (linear_f8_tc.cu).
int linear_f8_tc(const char *fn, const F8Args &a, cudaStream_t st);

}  // namespace sxb
