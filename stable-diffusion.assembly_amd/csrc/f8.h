// MUL_MAT of 8-bit floating-point weights (E4M3) with a scale for each block of
// 128 x 128 (f8.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "device.h"

namespace sdhip {

constexpr int64_t kF8Block = 128;

// y[m][n] = sum_k x[m][k] w[n][k] scales[n / 128][k / 128] and its chain, x held in
// E4M3 by groups of 128 of K, or with `half` the gated GELU of it: y[m][j] = P[m][j]
// GELU(P[m][half + j]).
struct F8Args {
    const float *x;
    int64_t ldx;
    const uint8_t *w;
    int64_t row_bytes;
    const float *scales;
    int64_t ld_scales;
    float *y;  // the output, or the redirect, or the gated output
    int64_t ldy;
    int64_t M, N, K;
    int64_t ne1, ne2;  // the output's rows and matrices, for the chain's coordinates
    int64_t half;      // gated: N / 2; else 0
    int32_t from_redirect;
    DevChain chain;
};

// The work buffer of a product (gated or not) of M rows; `whole`, whether the
// weights' rows are of whole 16 bytes at multiples of them.
size_t f8_work_size(int64_t M, int64_t N, int64_t K, bool whole);
hipError_t launch_f8_mul_mat(const F8Args &a, bool whole, void *work, hipStream_t stream);

}  // namespace sdhip
