// Rotary positions of several axes after the heads' norm: which calls are taken,
// and the launch.

#include <hip/hip_runtime.h>

#include <cmath>

#include "host.h"
#include "rope.h"

namespace sdhip {

namespace {

// Strides of 0 or more: what a tensor reaches lies behind its data.
bool forward(const sdhip_tensor *t) {
    return t == nullptr || (t->nb[0] >= 0 && t->nb[1] >= 0 && t->nb[2] >= 0 && t->nb[3] >= 0);
}

// Rows of `size` bytes a number: nb[0] that, the others any multiple of it, at
// such an address.
bool rows_of(const sdhip_tensor *t, int64_t size) {
    return t->nb[0] == size && t->nb[1] % size == 0 && t->nb[2] % size == 0 && t->nb[3] % size == 0 && forward(t) &&
           reinterpret_cast<uintptr_t>(t->data) % static_cast<uintptr_t>(size) == 0;
}

// The sum of the axes' numbers, or -1 where they are none that are taken.
int64_t turned_of(const sdhip_rope_axes *axes, int64_t d) {
    if (axes->count < 1 || axes->count > SDHIP_MAX_AXES) return -1;
    if (axes->order != SDHIP_ROPE_ADJACENT && axes->order != SDHIP_ROPE_HALVES) return -1;
    int64_t n = 0;
    for (int a = 0; a < axes->count; ++a) {
        if (axes->dims[a] < 2 || axes->dims[a] % 2 != 0 || !(axes->base[a] > 0.0f) || !std::isfinite(axes->base[a])) return -1;
        n += axes->dims[a];
    }
    return n <= d ? n : -1;
}

}  // namespace

}  // namespace sdhip

using namespace sdhip;

extern "C" {

int sdhip_rope_supported(const sdhip_tensor *x, const sdhip_row_norm *norm, const sdhip_tensor *positions,
                         const sdhip_rope_axes *axes, const sdhip_tensor *y) {
    if (x == nullptr || positions == nullptr || axes == nullptr || y == nullptr) return 0;
    if (x->ne[0] > kRopeMost || !same_shape(x, y)) return 0;
    for (int k = 0; k < 4; ++k) {
        if (x->ne[k] < 1 || x->ne[k] > INT32_MAX) return 0;
    }
    // Heads are counted in 32 bits, tokens, and parts of their heads, in 64.
    if (x->ne[2] > (int64_t{1} << 24) || x->ne[1] > (int64_t{1} << 40) / x->ne[3]) return 0;
    if (!holds_f32(x) || !rows_of(x, 4)) return 0;
    if (!(holds_f32(y) && rows_of(y, 4)) && !(holds_f16(y) && rows_of(y, 2))) return 0;
    if (turned_of(axes, x->ne[0]) < 0 || !row_norm_taken(norm, x)) return 0;
    if (norm != nullptr && (!forward(norm->weight) || !forward(norm->bias))) return 0;
    if (!holds_f32(positions) || !rows_of(positions, 4) || positions->ne[0] != axes->count ||
        (positions->ne[1] != x->ne[1] && positions->ne[1] != 1) || positions->ne[2] != 1 ||
        (positions->ne[3] != x->ne[3] && positions->ne[3] != 1)) {
        return 0;
    }
    if (!elements_apart(y)) return 0;
    if (!(y->data == x->data && same_layout(x, y)) && tensors_share(x, y)) return 0;
    return !tensors_share(positions, y) && (norm == nullptr || (!tensors_share(norm->weight, y) && !tensors_share(norm->bias, y)));
}

sdhip_status sdhip_rope(const sdhip_tensor *x, const sdhip_row_norm *norm, const sdhip_tensor *positions,
                        const sdhip_rope_axes *axes, const sdhip_tensor *y, void *stream) {
    if (!sdhip_rope_supported(x, norm, positions, axes, y)) return fail(SDHIP_UNSUPPORTED, "rope: operands not taken");
    const sdhip_tensor *const all[] = {x, positions, y, norm != nullptr ? norm->weight : nullptr,
                                       norm != nullptr ? norm->bias : nullptr};
    for (const sdhip_tensor *t : all) {
        if (t != nullptr && t->data == nullptr) return fail(SDHIP_ERROR, "rope: a tensor without data");
    }
    RopeArgs a{};
    a.x = static_cast<const float *>(x->data);
    a.y = y->data;
    a.positions = static_cast<const float *>(positions->data);
    a.half = y->type == SDHIP_TYPE_F16;
    for (int k = 0; k < 4; ++k) {
        // Along an extent of 1 there is nothing to step over.
        a.xnb[k] = x->ne[k] == 1 ? 0 : x->nb[k] / 4;
        a.ynb[k] = y->ne[k] == 1 ? 0 : y->nb[k] / y->nb[0];
    }
    a.pnb1 = positions->ne[1] == 1 ? 0 : positions->nb[1] / 4;
    a.pnb3 = positions->ne[3] == 1 ? 0 : positions->nb[3] / 4;
    a.d = static_cast<int32_t>(x->ne[0]);
    a.tokens = x->ne[1];
    a.heads = static_cast<int32_t>(x->ne[2]);
    a.batch = x->ne[3];
    a.order = axes->order;
    a.turned = static_cast<int32_t>(turned_of(axes, x->ne[0]));
    a.count = axes->count;
    for (int i = 0; i < axes->count; ++i) {
        a.first[i + 1] = a.first[i] + axes->dims[i] / 2;
        a.from[i] = axes->shared ? 0 : a.first[i];
        a.rate[i] = -2.0 * std::log2(static_cast<double>(axes->base[i])) / (axes->shared ? a.turned : axes->dims[i]);
    }
    a.inverse = 1.0 / static_cast<double>(a.d);
    a.norm = row_norm(norm);
    return launched(launch_rope(a, static_cast<hipStream_t>(stream)), "rope");
}

}  // extern "C"
