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

// A written tensor: apart in itself, and in no byte range that is read, but
// for y's or residual's own memory in the same layout.
bool written(const sdhip_tensor *t, const sdhip_tensor *const *rows, const sdhip_tensor *const *operands, int count) {
    if (!elements_apart(t)) return false;
    for (int i = 0; i < 2; ++i) {
        if (rows[i] != nullptr && !(t->data == rows[i]->data && same_layout(t, rows[i])) && tensors_share(t, rows[i])) {
            return false;
        }
    }
    for (int i = 0; i < count; ++i) {
        if (tensors_share(t, operands[i])) return false;
    }
    return true;
}

void strides_of(const sdhip_tensor *t, int64_t (&nb)[4]) {
    for (int k = 0; k < 4; ++k) nb[k] = t != nullptr ? t->nb[k] / 4 : 0;
}

}  // namespace

RowOperand row_operand(const sdhip_tensor *t) {
    RowOperand o{};
    if (t == nullptr) return o;
    o.data = static_cast<const float *>(t->data);
    for (int k = 0; k < 4; ++k) o.nb[k] = t->ne[k] == 1 ? 0 : t->nb[k] / 4;
    return o;
}

RowNorm row_norm(const sdhip_row_norm *n) {
    RowNorm r{};
    if (n == nullptr) return r;
    r.kind = n->kind;
    r.eps = n->eps;
    r.offset = n->weight_offset;
    r.weight = row_operand(n->weight);
    r.bias = row_operand(n->bias);
    return r;
}

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
    if (!row_norm_taken(post, residual) || !row_norm_taken(pre, residual) || (gate != nullptr && !broadcasts(gate, residual))) {
        return 0;
    }
    const sdhip_tensor *const inputs[] = {y, residual};
    const sdhip_tensor *const operands[] = {gate, post != nullptr ? post->weight : nullptr,
                                            post != nullptr ? post->bias : nullptr,
                                            pre != nullptr ? pre->weight : nullptr,
                                            pre != nullptr ? pre->bias : nullptr};
    if (sum != nullptr && !written(sum, inputs, operands, 5)) return 0;
    if (out != nullptr && !written(out, inputs, operands, 5)) return 0;
    return !tensors_share(sum, out);
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
    a.post = row_norm(post);
    a.pre = row_norm(pre);
    a.gate = row_operand(gate);
    return launched(launch_norm_residual(a, static_cast<hipStream_t>(stream)), "norm_residual");
}

}  // extern "C"
