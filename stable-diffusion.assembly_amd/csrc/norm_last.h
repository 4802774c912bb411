// GROUP_NORM of channels-last tensors (norm_last.hip).  Strides in elements.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "device.h"

namespace sdhip {

struct GroupNormLastArgs {
    const float *x;
    float *y;
    int64_t channels, width, pixels, images;
    int64_t xpixel, ximage, ypixel, yimage;  // from one pixel, or image, to the next
    int64_t groups, per_group;               // groups of an image that have channels; channels of a group
    float eps;
    DevChain chain;
    // How it is split (group_norm_last_shape).
    int64_t image0;              // the launch's first image
    int32_t slab_groups, slabs;  // groups of a workgroup's channels; of those in an image
    int32_t chunks;              // of an image's pixels, a workgroup each
    int32_t parts;               // the chunks that sums were taken over
    int64_t chunk;               // pixels
    double *partials;            // [image][group][part][2]: sums of x - c and of its squares, c the group's first number
    double *firsts;              // [image][group]: c
};

// The extents of a call, for its split and its work buffer.
struct GroupNormLastShape {
    int64_t channels, pixels, images, groups, per_group;
};

size_t group_norm_last_work_size(const GroupNormLastShape &s);
hipError_t launch_group_norm_last(GroupNormLastArgs a, void *work, hipStream_t stream);

}  // namespace sdhip
