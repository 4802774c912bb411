// The norms after and before a block with its gate and residual (residual.hip).
// Strides in elements.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device.h"

namespace sdhip {

// A tensor broadcast over the rows: strides 0 along what it is broadcast
// over; null where there is none.
struct RowOperand {
    const float *data;
    int64_t nb[4];
};

struct RowNorm {
    int32_t kind;  // SDHIP_ROW_NORM_*
    float eps, offset;
    RowOperand weight, bias;
};

struct ResidualArgs {
    const float *y;  // or null
    const float *residual;
    float *sum;  // or null
    float *out;  // or null
    int64_t ynb[4], rnb[4], snb[4], onb[4];
    int64_t ne0, ne1, ne2, rows;
    int64_t first;  // the launch's first row
    double inverse;  // 1 / ne0
    float branch_scale, residual_scale;
    RowNorm post, pre;
    RowOperand gate;
};

hipError_t launch_norm_residual(const ResidualArgs &a, hipStream_t stream);

}  // namespace sdhip
