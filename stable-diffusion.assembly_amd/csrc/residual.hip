// The norms after and before a transformer block with its gate and residual:
//     z = post(y),  s = residual_scale residual + branch_scale (gate z),  n = pre(s),
// a row's norm by its mean and the mean of its squares about it (LAYER), or
// about 0 (RMS), both summed in double: no square of a single-precision
// number passes it, and the mean is held in two single-precision parts.

#include "host.h"
#include "profile.h"
#include "residual.h"

namespace sdhip {

namespace {

constexpr int kThreads = 256;

struct Place {
    int64_t i1, i2, i3;
};

__device__ __forceinline__ int64_t row_at(const int64_t (&nb)[4], const Place &p) {
    return p.i1 * nb[1] + p.i2 * nb[2] + p.i3 * nb[3];
}

// What a norm does to the numbers of a row: (v - hi - lo) scale.
struct Moments {
    float hi, lo, scale;
};

__device__ __forceinline__ Moments moments(int32_t kind, double mean, double squares, double n, float eps) {
    Moments m{0.0f, 0.0f, 1.0f};
    if (kind == SDHIP_ROW_NORM_LAYER) {
        m.hi = static_cast<float>(mean);
        m.lo = static_cast<float>(mean - static_cast<double>(m.hi));
    }
    if (kind != SDHIP_ROW_NORM_NONE) m.scale = static_cast<float>(1.0 / sqrt(squares / n + static_cast<double>(eps)));
    return m;
}

__device__ __forceinline__ float normed(float v, const Moments &m) { return __fmul_rn(v - m.hi - m.lo, m.scale); }

__device__ __forceinline__ double block_sum(double v, double *lds) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
    for (uint32_t w = 0; w < blockDim.x / 64; ++w) s += lds[w];
    return s;
}

// A row a workgroup, read again for each of its sums: rows of any length.
__global__ __launch_bounds__(kThreads) void norm_residual_long_kernel(ResidualArgs a) {
    __shared__ double lds[kThreads / 64];
    const int64_t row = blockIdx.x;
    const Place p{row % a.ne1, (row / a.ne1) % a.ne2, row / (a.ne1 * a.ne2)};
    const float *y = a.y != nullptr ? a.y + row_at(a.ynb, p) : nullptr;
    const float *r = a.residual + row_at(a.rnb, p);
    float *sum = a.sum != nullptr ? a.sum + row_at(a.snb, p) : nullptr;
    float *out = a.out != nullptr ? a.out + row_at(a.onb, p) : nullptr;
    const double n = static_cast<double>(a.ne0);
    const auto stats = [&](int32_t kind, float eps, auto value) {
        double mean = 0.0, squares = 0.0;
        if (kind == SDHIP_ROW_NORM_LAYER) {
            double s = 0.0;
            for (int64_t i = threadIdx.x; i < a.ne0; i += kThreads) s += static_cast<double>(value(i));
            mean = block_sum(s, lds) / n;
        }
        if (kind != SDHIP_ROW_NORM_NONE) {
            double s = 0.0;
            for (int64_t i = threadIdx.x; i < a.ne0; i += kThreads) {
                const double d = static_cast<double>(value(i)) - mean;
                s += d * d;
            }
            squares = block_sum(s, lds);
        }
        return moments(kind, mean, squares, n, eps);
    };
    const auto affine = [&](const RowNorm &w, float v, int64_t i) {
        if (w.weight.data != nullptr) {
            v = __fmul_rn(v, __fadd_rn(w.weight.data[row_at(w.weight.nb, p) + i * w.weight.nb[0]], w.offset));
        }
        if (w.bias.data != nullptr) v = __fadd_rn(v, w.bias.data[row_at(w.bias.nb, p) + i * w.bias.nb[0]]);
        return v;
    };
    Moments post{0.0f, 0.0f, 1.0f};
    if (y != nullptr) post = stats(a.post.kind, a.post.eps, [&](int64_t i) { return y[i]; });
    const auto joined = [&](int64_t i) {
        float s = __fmul_rn(a.residual_scale, r[i]);
        if (y == nullptr) return s;
        float z = affine(a.post, a.post.kind != SDHIP_ROW_NORM_NONE ? normed(y[i], post) : y[i], i);
        if (a.gate.data != nullptr) z = __fmul_rn(z, a.gate.data[row_at(a.gate.nb, p) + i * a.gate.nb[0]]);
        return __fadd_rn(s, __fmul_rn(a.branch_scale, z));
    };
    // With sum in place of y or of residual a number is read and then
    // written by one thread, and from here on read from sum.
    if (sum != nullptr) {
        for (int64_t i = threadIdx.x; i < a.ne0; i += kThreads) sum[i] = joined(i);
    }
    if (out == nullptr) return;
    const auto value = [&](int64_t i) { return sum != nullptr ? sum[i] : joined(i); };
    const Moments pre = stats(a.pre.kind, a.pre.eps, value);
    for (int64_t i = threadIdx.x; i < a.ne0; i += kThreads) {
        const float v = value(i);
        out[i] = affine(a.pre, a.pre.kind != SDHIP_ROW_NORM_NONE ? normed(v, pre) : v, i);
    }
}

}  // namespace

hipError_t launch_norm_residual(const ResidualArgs &a, hipStream_t stream) {
    KernelScope scope("norm_residual", stream);
    SDHIP_LAUNCH(norm_residual_long_kernel, dim3(static_cast<uint32_t>(a.rows)), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace sdhip
