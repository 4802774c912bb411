// GROUP_NORM of channels-last tensors (norm_last.hip).  Strides in elements.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "device.h"

namespace sdhip {

// The steps of a chain that is some of these, in this order, by one number a channel.
enum : int32_t { kPlainMul = 1, kPlainAdd = 2, kPlainSilu = 4 };

struct GroupNormLastArgs {
    const float *x;
    float *y;
    int64_t channels, width, pixels, images;
    int64_t xpixel, ximage, ypixel, yimage;  // from one pixel, or image, to the next
    int64_t groups, per_group;               // groups of an image that have channels; channels of a group
    float eps;
    DevChain chain;
    int32_t plain;  // its steps, where it is such a chain; else 0
    // A launch's workgroups: from image0 on, slab_groups groups' channels and `chunk`
    // pixels each, `chunks` of an image.
    int64_t image0, chunk;
    int32_t slab_groups, slabs, chunks;
    int32_t parts;     // the chunks that sums were taken over
    double *partials;  // [image][group][part][2]: sums of x - c and of its squares, c the group's first number
    double *firsts;    // [image][group]: c
    double *joined;    // [image][group][2]: the mean, and what x less it is multiplied by; or null
};

// The extents of a call, for its split and its work buffer.
struct GroupNormLastShape {
    int64_t channels, pixels, images, groups, per_group;
};

size_t group_norm_last_work_size(const GroupNormLastShape &s);
hipError_t launch_group_norm_last(GroupNormLastArgs a, void *work, hipStream_t stream);

}  // namespace sdhip
