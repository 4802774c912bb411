// GROUP_NORM of channels-last tensors: which calls are taken, and the launch.

#include <hip/hip_runtime.h>

#include "host.h"
#include "norm_last.h"

namespace sdhip {

namespace {

// Images of evenly spaced pixels, their channels side by side.
bool pixels_of(const sdhip_tensor *t) {
    int64_t row;
    return holds_f32(t) && t->nb[1] % 4 == 0 && t->nb[2] % 4 == 0 && t->nb[3] % 4 == 0 && t->nb[1] >= 0 && t->nb[2] >= 0 &&
           t->nb[3] >= 0 &&
           reinterpret_cast<uintptr_t>(t->data) % 4 == 0 &&
           (t->ne[1] == 1 || t->ne[2] == 1 || (!__builtin_mul_overflow(t->nb[1], t->ne[1], &row) && t->nb[2] == row));
}

int64_t pixel_stride(const sdhip_tensor *t) { return (t->ne[1] > 1 ? t->nb[1] : t->ne[2] > 1 ? t->nb[2] : 0) / 4; }

GroupNormLastShape shape_of(const sdhip_tensor *x, int groups) {
    const int64_t per_group = ceil_div(x->ne[0], groups);
    return {x->ne[0], x->ne[1] * x->ne[2], x->ne[3], ceil_div(x->ne[0], per_group), per_group};
}

}  // namespace

}  // namespace sdhip

using namespace sdhip;

extern "C" {

int sdhip_group_norm_last_supported(const sdhip_tensor *x, const sdhip_tensor *y, int groups) {
    if (x == nullptr || y == nullptr || groups < 1 || !same_shape(x, y)) return 0;
    // Channels, pixels and images are counted in 32 bits, all numbers in 64.
    constexpr int64_t kChannels = int64_t{1} << 24, kNumbers = int64_t{1} << 40;
    for (int k = 0; k < 4; ++k) {
        if (x->ne[k] < 1 || x->ne[k] > INT32_MAX) return 0;
    }
    if (x->ne[0] > kChannels || x->ne[1] > INT32_MAX / x->ne[2]) return 0;
    if (x->ne[1] * x->ne[2] > kNumbers / x->ne[0] / x->ne[3]) return 0;
    if (!pixels_of(x) || !pixels_of(y) || !elements_apart(y)) return 0;
    return (y->data == x->data && same_layout(x, y)) || !tensors_share(x, y);
}

size_t sdhip_group_norm_last_work_size(const sdhip_tensor *x, const sdhip_tensor *y, int groups) {
    if (!sdhip_group_norm_last_supported(x, y, groups)) return 0;
    return group_norm_last_work_size(shape_of(x, groups));
}

sdhip_status sdhip_group_norm_last(const sdhip_tensor *x, const sdhip_tensor *y, int groups, float eps,
                                   const sdhip_epilogue *chain, void *work, size_t work_size, void *stream) {
    if (!sdhip_group_norm_last_supported(x, y, groups)) {
        return fail(SDHIP_UNSUPPORTED, "group_norm_last: operands not taken");
    }
    if (chain != nullptr && chain->redirect != nullptr) {
        return fail(SDHIP_UNSUPPORTED, "group_norm_last: no residual redirect after a normalisation");
    }
    if (x->data == nullptr || y->data == nullptr) return fail(SDHIP_ERROR, "group_norm_last: a tensor without data");
    ChainRun run;
    sdhip_status s = chain_plan(y, chain, run);
    if (s != SDHIP_OK) return s;
    if (!chain_apart(y, chain)) return fail(SDHIP_UNSUPPORTED, "group_norm_last: the output overlaps a chain operand");
    const GroupNormLastShape shape = shape_of(x, groups);
    const size_t need = group_norm_last_work_size(shape);
    if (const sdhip_status ws = check_work("group_norm_last", work, work_size, need); ws != SDHIP_OK) return ws;
    GroupNormLastArgs a{};
    a.chain = run.fused;
    a.x = static_cast<const float *>(x->data);
    a.y = static_cast<float *>(y->data);
    a.channels = shape.channels;
    a.width = x->ne[1];
    a.pixels = shape.pixels;
    a.images = shape.images;
    a.xpixel = pixel_stride(x);
    a.ypixel = pixel_stride(y);
    a.ximage = x->ne[3] > 1 ? x->nb[3] / 4 : 0;
    a.yimage = y->ne[3] > 1 ? y->nb[3] / 4 : 0;
    a.groups = shape.groups;
    a.per_group = shape.per_group;
    a.eps = eps;
    s = launched(launch_group_norm_last(a, work, static_cast<hipStream_t>(stream)), "group_norm_last");
    return s == SDHIP_OK ? chain_after(run, static_cast<hipStream_t>(stream)) : s;
}

}  // extern "C"
