// Rotary positions of several axes after the heads' norm (rope.hip).  Strides in
// elements.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device.h"
#include "row_norm.h"

namespace sdhip {

constexpr int kRopeMost = 512;  // numbers of a head

struct RopeArgs {
    const float *x;
    void *y;  // single precision, or with `half` FP16
    const float *positions;
    int64_t xnb[4], ynb[4];
    int64_t pnb1, pnb3;  // positions' strides along the tokens and the batch; 0 where broadcast
    int64_t tokens, batch;
    int32_t d, heads, half;
    int32_t order;               // SDHIP_ROPE_*
    int32_t turned;              // numbers of a head in pairs: n
    int32_t count;
    int32_t first[SDHIP_MAX_AXES + 1];  // an axis's first pair; n / 2 past the last
    int32_t from[SDHIP_MAX_AXES];       // the pair that an axis's frequencies count from
    double rate[SDHIP_MAX_AXES];        // the frequency of pair p is 2^(rate (p - from))
    double inverse;                     // 1 / d
    RowNorm norm;
    int32_t parts;  // of a token's heads, a wave each
};

hipError_t launch_rope(RopeArgs a, hipStream_t stream);

}  // namespace sdhip
