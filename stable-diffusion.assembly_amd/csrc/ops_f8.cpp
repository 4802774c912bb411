// MUL_MAT and MUL_MAT with the gated GELU of weights in 8-bit floating point with
// a scale for each block of 128 x 128: which calls are taken, and the launch.

#include <hip/hip_runtime.h>

#include "f8.h"
#include "host.h"

namespace sdhip {

namespace {

bool holds_f8(const sdhip_tensor *t) { return t != nullptr && t->type == SDHIP_TYPE_F8_E4M3 && t->nb[0] == 1; }

F8Args args_of(const sdhip_tensor *w, const sdhip_tensor *scales, const sdhip_tensor *x, const sdhip_tensor *y) {
    F8Args a{};
    a.x = static_cast<const float *>(x->data);
    a.ldx = x->nb[1] / 4;
    a.w = static_cast<const uint8_t *>(w->data);
    a.row_bytes = w->nb[1];
    a.scales = static_cast<const float *>(scales->data);
    a.ld_scales = scales->nb[1] / 4;
    a.K = w->ne[0];
    a.N = w->ne[1];
    a.M = x->ne[1] * x->ne[2] * x->ne[3];
    a.ne1 = y->ne[1];
    a.ne2 = y->ne[2];
    a.ldy = y->nb[1] / 4;
    return a;
}

// Whether rows of the weights are of whole 16 bytes at multiples of them, 128 rows
// within 32 bits.
bool whole(const sdhip_tensor *w) {
    return w->ne[0] % 16 == 0 && w->nb[1] % 16 == 0 && w->nb[1] <= (int64_t{1} << 24) &&
           reinterpret_cast<uintptr_t>(w->data) % 16 == 0;
}

bool whole_floats(const sdhip_tensor *t) { return reinterpret_cast<uintptr_t>(t->data) % 4 == 0; }

sdhip_status misaligned(const char *what) {
    return fail(SDHIP_ERROR, "%s: single precision at an address that is no multiple of 4", what);
}

// The product into a.y, `columns` wide, which what it reads shares no byte with.
sdhip_status product(const F8Args &a, const sdhip_tensor *w, const sdhip_tensor *scales, const sdhip_tensor *x,
                     int64_t columns, void *work, size_t work_size, hipStream_t stream, const char *what) {
    if (w->data == nullptr || scales->data == nullptr || x->data == nullptr || a.y == nullptr) {
        return fail(SDHIP_ERROR, "%s: a tensor without data", what);
    }
    if (!whole_floats(x) || !whole_floats(scales) || reinterpret_cast<uintptr_t>(a.y) % 4 != 0) return misaligned(what);
    const size_t on = static_cast<size_t>((a.M - 1) * a.ldy + columns) * 4;
    for (const sdhip_tensor *t : {w, scales, x}) {
        if (spans_overlap(a.y, on, t->data, tensor_span(t))) {
            return fail(SDHIP_ERROR, "%s: the output lies over an operand", what);
        }
    }
    const size_t need = f8_work_size(a.M, a.N, a.K, whole(w));
    if (const sdhip_status ws = check_work(what, work, work_size, need); ws != SDHIP_OK) return ws;
    return launched(launch_f8_mul_mat(a, whole(w), work, stream), what);
}

}  // namespace

}  // namespace sdhip

using namespace sdhip;

extern "C" {

int sdhip_mul_mat_f8_supported(const sdhip_tensor *w, const sdhip_tensor *scales, const sdhip_tensor *x,
                               const sdhip_tensor *y) {
    if (w == nullptr || scales == nullptr || x == nullptr || y == nullptr) return 0;
    // Extents to what a launch counts, 2^32 threads, and what it divides in 32 bits.
    constexpr int64_t kMost = int64_t{1} << 25, kWeights = int64_t{1} << 36, kOutputs = int64_t{1} << 35;
    constexpr int64_t kNumbers = int64_t{1} << 37;
    if (!holds_f8(w) || w->ne[0] < 1 || w->ne[0] > INT32_MAX - kF8Block || w->ne[1] < 1 || w->ne[1] > kMost ||
        w->ne[1] > kWeights / w->ne[0] || w->ne[2] != 1 || w->ne[3] != 1 || w->nb[1] < w->ne[0]) {
        return 0;
    }
    const int64_t k_blocks = ceil_div(w->ne[0], kF8Block);
    if (!holds_f32(scales) || scales->ne[0] != k_blocks || scales->ne[1] != ceil_div(w->ne[1], kF8Block) ||
        scales->ne[2] != 1 || scales->ne[3] != 1 || scales->nb[1] % 4 != 0 || scales->nb[1] < 4 * k_blocks) {
        return 0;
    }
    int64_t rows = 1;
    for (int k = 1; k < 4; ++k) {
        if (x->ne[k] < 1 || x->ne[k] > kMost || y->ne[k] != x->ne[k]) return 0;
        rows *= x->ne[k];
        if (rows > kMost) return 0;
    }
    if (w->ne[1] > kOutputs / rows || kF8Block * k_blocks > kNumbers / rows) return 0;
    return x->ne[0] == w->ne[0] && y->ne[0] == w->ne[1] && holds_f32(x) && contiguous(x) && holds_f32(y) && contiguous(y);
}

size_t sdhip_mul_mat_f8_work_size(const sdhip_tensor *w, const sdhip_tensor *scales, const sdhip_tensor *x,
                                  const sdhip_tensor *y) {
    if (!sdhip_mul_mat_f8_supported(w, scales, x, y)) return 0;
    return f8_work_size(x->ne[1] * x->ne[2] * x->ne[3], w->ne[1], w->ne[0], whole(w));
}

sdhip_status sdhip_mul_mat_f8(const sdhip_tensor *w, const sdhip_tensor *scales, const sdhip_tensor *x,
                              const sdhip_tensor *y, const sdhip_epilogue *chain, void *work, size_t work_size,
                              void *stream) {
    if (!sdhip_mul_mat_f8_supported(w, scales, x, y)) return fail(SDHIP_UNSUPPORTED, "mul_mat_f8: operands not taken");
    ChainRun run;
    sdhip_status s = chain_plan(y, chain, run);
    if (s != SDHIP_OK) return s;
    if (!chain_apart(y, chain)) return fail(SDHIP_UNSUPPORTED, "mul_mat_f8: the output overlaps a chain operand");
    if (chain != nullptr && chain->redirect != nullptr && !whole_floats(chain->redirect)) return misaligned("mul_mat_f8");
    for (const sdhip_tensor *t : {w, scales, x}) {
        if (chain != nullptr && tensors_share(chain->redirect, t)) return fail(SDHIP_ERROR, "mul_mat_f8: the output lies over an operand");
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    F8Args a = args_of(w, scales, x, y);
    a.chain = run.fused;
    a.y = run.out;
    a.from_redirect = run.from_redirect;
    s = product(a, w, scales, x, a.N, work, work_size, st, "mul_mat_f8");
    return s == SDHIP_OK ? chain_after(run, st) : s;
}

int sdhip_mul_mat_f8_gated_supported(const sdhip_tensor *w, const sdhip_tensor *scales, const sdhip_tensor *x,
                                     const sdhip_tensor *y, const sdhip_tensor *out) {
    if (!sdhip_mul_mat_f8_supported(w, scales, x, y) || out == nullptr || y->ne[0] % 2 != 0) return 0;
    if (!holds_f32(out) || !contiguous(out) || out->ne[0] != y->ne[0] / 2) return 0;
    for (int k = 1; k < 4; ++k) {
        if (out->ne[k] != y->ne[k]) return 0;
    }
    // What the result is written to is not what the product reads, nor the
    // product's own place.
    for (const sdhip_tensor *t : {w, scales, x, y}) {
        if (tensors_share(out, t)) return 0;
    }
    return 1;
}

sdhip_status sdhip_mul_mat_f8_gated(const sdhip_tensor *w, const sdhip_tensor *scales, const sdhip_tensor *x,
                                    const sdhip_tensor *y, const sdhip_epilogue *chain, const sdhip_tensor *out,
                                    void *work, size_t work_size, void *stream) {
    if (!sdhip_mul_mat_f8_gated_supported(w, scales, x, y, out)) {
        return fail(SDHIP_UNSUPPORTED, "mul_mat_f8_gated: operands not taken");
    }
    if (chain != nullptr && chain->redirect != nullptr) {
        return fail(SDHIP_UNSUPPORTED, "mul_mat_f8_gated: a chain with a residual redirect is not gated");
    }
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (out->data == nullptr) return fail(SDHIP_ERROR, "mul_mat_f8_gated: a tensor without data");
    if (!whole_floats(out)) return misaligned("mul_mat_f8_gated");
    if (tuning().fuse == 0) {
        // The gated GELU apart: the product and its chain into y, then out from
        // y's halves.
        const sdhip_status s = sdhip_mul_mat_f8(w, scales, x, y, chain, work, work_size, stream);
        if (s != SDHIP_OK) return s;
        return gated_after(static_cast<const float *>(y->data), static_cast<float *>(out->data),
                           x->ne[1] * x->ne[2] * x->ne[3], y->ne[0] / 2, y->nb[1] / 4, out->nb[1] / 4, st);
    }
    F8Args a = args_of(w, scales, x, y);
    const sdhip_status s = device_chain(chain, y->ne, a.chain);
    if (s != SDHIP_OK) return s;
    for (int i = 0; chain != nullptr && i < chain->count; ++i) {
        if (chain->steps[i].kind != SDHIP_STEP_SILU && tensors_share(out, &chain->steps[i].operand)) {
            return fail(SDHIP_UNSUPPORTED, "mul_mat_f8_gated: the output overlaps a chain operand");
        }
    }
    a.y = static_cast<float *>(out->data);
    a.ldy = out->nb[1] / 4;
    a.half = y->ne[0] / 2;
    return product(a, w, scales, x, a.half, work, work_size, st, "mul_mat_f8_gated");
}

}  // extern "C"
