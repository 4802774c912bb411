// MUL_MAT of 4-bit weights in blocks of 32 along K (q4.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "device.h"

namespace sdhip {

// y[m][n] = sum_k x[m][k] w[n][k] and its chain, or with `half` the gated GELU
// of it: y[m][j] = P[m][j] GELU(P[m][half + j]).  The weights are rows of
// K / 32 blocks, `row_bytes` apart, an even number at an even address; with
// `least`, Q4_1's blocks of 20 bytes, else Q4_0's of 18.
struct Q4Args {
    const float *x;
    int64_t ldx;
    const uint8_t *w;
    int64_t row_bytes;
    int32_t least;
    int32_t from_redirect;
    float *y;  // the output, or the redirect, or the gated output
    int64_t ldy;
    int64_t M, N, K;
    int64_t ne1, ne2;  // the output's rows and matrices, for the chain's coordinates
    int64_t half;      // gated: N / 2; else 0
    DevChain chain;
};

// The work buffer of a product (gated or not) of M rows: its operands as the
// kernels read them; 0 for few rows.
size_t q4_work_size(int64_t M, int64_t N, int64_t K, bool least);
hipError_t launch_q4_mul_mat(const Q4Args &a, void *work, hipStream_t stream);

}  // namespace sdhip
