// The norms after and before a block with its gate and residual: which calls
// are taken, and the launch.

#include <hip/hip_runtime.h>

#include "host.h"
#include "residual.h"

namespace sdhip {

namespace {

// Rows of single precision: nb[0] = 4, the others any multiple of 4 (which
// need not be those of an array without holes).
bool rows_of(const sdhip_tensor *t, const sdhip_tensor *shape) {
    return holds_f32(t) && same_shape(t, shape) && t->nb[1] % 4 == 0 && t->nb[2] % 4 == 0 && t->nb[3] % 4 == 0 &&
           reinterpret_cast<uintptr_t>(t->data) % 4 == 0;
}

bool broadcast(const sdhip_tensor *t, const sdhip_tensor *shape) {
    if (!holds_f32(t) || reinterpret_cast<uintptr_t>(t->data) % 4 != 0) return false;
    for (int k = 0; k < 4; ++k) {
        if ((t->ne[k] != shape->ne[k] && t->ne[k] != 1) || t->nb[k] % 4 != 0) return false;
    }
    return true;
}

bool norm_taken(const sdhip_row_norm *n, const sdhip_tensor *shape) {
    if (n == nullptr) return true;
    return n->kind >= SDHIP_ROW_NORM_NONE && n->kind <= SDHIP_ROW_NORM_RMS &&
           (n->weight == nullptr || broadcast(n->weight, shape)) && (n->bias == nullptr || broadcast(n->bias, shape));
}

// Whether no two numbers of t lie in one place: along the dimensions in the
// order of their strides each step passes all that the ones before it reach.
bool apart(const sdhip_tensor *t) {
    int64_t reach = 4;
    bool done[4] = {};
    for (int pass = 0; pass < 4; ++pass) {
        int next = -1;
        for (int k = 0; k < 4; ++k) {
            if (!done[k] && (next < 0 || t->nb[k] < t->nb[next])) next = k;
        }
        done[next] = true;
        if (t->ne[next] == 1) continue;
        if (t->nb[next] < reach) return false;
        if (t->nb[next] > INT64_MAX / t->ne[next]) return false;
        reach = t->nb[next] * t->ne[next];
    }
    return true;
}

bool share(const sdhip_tensor *a, const sdhip_tensor *b) {
    return a != nullptr && b != nullptr && spans_overlap(a->data, tensor_span(a), b->data, tensor_span(b));
}

// A written tensor: apart in itself, and in no byte range that is read, but
// for y's or residual's own memory in the same layout.
bool written(const sdhip_tensor *t, const sdhip_tensor *const *rows, const sdhip_tensor *const *operands, int count) {
    if (!apart(t)) return false;
    for (int i = 0; i < 2; ++i) {
        if (rows[i] != nullptr && !(t->data == rows[i]->data && same_layout(t, rows[i])) && share(t, rows[i])) {
            return false;
        }
    }
    for (int i = 0; i < count; ++i) {
        if (share(t, operands[i])) return false;
    }
    return true;
}

RowOperand operand_of(const sdhip_tensor *t) {
    RowOperand o{};
    if (t == nullptr) return o;
    o.data = static_cast<const float *>(t->data);
    for (int k = 0; k < 4; ++k) o.nb[k] = t->ne[k] == 1 ? 0 : t->nb[k] / 4;
    return o;
}

RowNorm norm_of(const sdhip_row_norm *n) {
    RowNorm r{};
    if (n == nullptr) return r;
    r.kind = n->kind;
    r.eps = n->eps;
    r.offset = n->weight_offset;
    r.weight = operand_of(n->weight);
    r.bias = operand_of(n->bias);
    return r;
}

void strides_of(const sdhip_tensor *t, int64_t (&nb)[4]) {
    for (int k = 0; k < 4; ++k) nb[k] = t != nullptr ? t->nb[k] / 4 : 0;
}

}  // namespace

}  // namespace sdhip

using namespace sdhip;

extern "C" {

int sdhip_norm_residual_supported(const sdhip_tensor *y, const sdhip_row_norm *post, const sdhip_tensor *gate,
                                  const sdhip_tensor *residual, const sdhip_tensor *sum, const sdhip_row_norm *pre,
                                  const sdhip_tensor *out) {
    if (residual == nullptr || (sum == nullptr && out == nullptr) || (pre == nullptr) != (out == nullptr)) return 0;
    if (y == nullptr && (post != nullptr || gate != nullptr)) return 0;
    // Rows, and the coordinates of one, are counted in 32 bits.
    int64_t rows = 1;
    for (int k = 0; k < 4; ++k) {
        if (residual->ne[k] < 1 || residual->ne[k] > INT32_MAX) return 0;
        if (k > 0) rows *= residual->ne[k];
        if (rows > INT32_MAX) return 0;
    }
    if (!rows_of(residual, residual)) return 0;
    const sdhip_tensor *const others[] = {y, sum, out};
    for (const sdhip_tensor *t : others) {
        if (t != nullptr && !rows_of(t, residual)) return 0;
    }
    if (!norm_taken(post, residual) || !norm_taken(pre, residual) || (gate != nullptr && !broadcast(gate, residual))) {
        return 0;
    }
    const sdhip_tensor *const inputs[] = {y, residual};
    const sdhip_tensor *const operands[] = {gate, post != nullptr ? post->weight : nullptr,
                                            post != nullptr ? post->bias : nullptr,
                                            pre != nullptr ? pre->weight : nullptr,
                                            pre != nullptr ? pre->bias : nullptr};
    if (sum != nullptr && !written(sum, inputs, operands, 5)) return 0;
    if (out != nullptr && !written(out, inputs, operands, 5)) return 0;
    return !share(sum, out);
}

sdhip_status sdhip_norm_residual(const sdhip_tensor *y, const sdhip_row_norm *post, const sdhip_tensor *gate,
                                 float branch_scale, const sdhip_tensor *residual, float residual_scale,
                                 const sdhip_tensor *sum, const sdhip_row_norm *pre, const sdhip_tensor *out,
                                 void *stream) {
    if (!sdhip_norm_residual_supported(y, post, gate, residual, sum, pre, out)) {
        return fail(SDHIP_UNSUPPORTED, "norm_residual: operands not taken");
    }
    const sdhip_tensor *const all[] = {y,
                                       gate,
                                       residual,
                                       sum,
                                       out,
                                       post != nullptr ? post->weight : nullptr,
                                       post != nullptr ? post->bias : nullptr,
                                       pre != nullptr ? pre->weight : nullptr,
                                       pre != nullptr ? pre->bias : nullptr};
    for (const sdhip_tensor *t : all) {
        if (t != nullptr && t->data == nullptr) return fail(SDHIP_ERROR, "norm_residual: a tensor without data");
    }
    ResidualArgs a{};
    a.y = y != nullptr ? static_cast<const float *>(y->data) : nullptr;
    a.residual = static_cast<const float *>(residual->data);
    a.sum = sum != nullptr ? static_cast<float *>(sum->data) : nullptr;
    a.out = out != nullptr ? static_cast<float *>(out->data) : nullptr;
    strides_of(y, a.ynb);
    strides_of(residual, a.rnb);
    strides_of(sum, a.snb);
    strides_of(out, a.onb);
    a.ne0 = residual->ne[0];
    a.inverse = 1.0 / static_cast<double>(a.ne0);
    a.ne1 = residual->ne[1];
    a.ne2 = residual->ne[2];
    a.rows = residual->ne[1] * residual->ne[2] * residual->ne[3];
    a.branch_scale = branch_scale;
    a.residual_scale = residual_scale;
    a.post = norm_of(post);
    a.pre = norm_of(pre);
    a.gate = operand_of(gate);
    return launched(launch_norm_residual(a, static_cast<hipStream_t>(stream)), "norm_residual");
}

}  // extern "C"
