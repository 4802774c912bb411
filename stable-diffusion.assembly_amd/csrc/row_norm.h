// A norm of rows of single precision (sdhip_row_norm) as kernels take it, and
// what they compute it with: a row's mean and the mean of its squares about it in
// double, brought to single precision once.  Strides in elements.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/sdhip.h"
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

// The host's descriptors as such operands (ops_residual.cpp).
RowOperand row_operand(const sdhip_tensor *t);
RowNorm row_norm(const sdhip_row_norm *n);

// What a norm does to the numbers of a row: (v power - hi - lo) scale, hi and lo
// of the mean times `power`: a power of two that keeps the differences within
// single precision, the mean's second part and `scale` normal numbers for rows of
// the greatest and of the least numbers (3e38 among -3e38 lies 4.5e38 from the
// mean; of numbers of 2^-140 a second part would be below 2^-149), else 1.
struct Moments {
    float hi, lo, scale, power;
};

// 1 / sqrt(v) within 2^-45 of itself: the hardware's, within 2^-24 or so, by one
// step of Newton's, a fifth of the operations of a root and a division (2 x 988
// rows of 2048 14.0 us, so 13.4; one of 4096 4.61 and 4.45).
__device__ __forceinline__ double inverse_root(double v) {
    const double r = __builtin_amdgcn_rsq(v);
    const double next = __builtin_fma(0.5 * r, __builtin_fma(-v * r, r, 1.0), r);
    return v > 0.0 && v < __builtin_inf() ? next : r;
}

// The mean of n numbers, of which `inverse` is 1 / n: exact where it is a double,
// by what the rounded quotient leaves of the sum, so that nothing is left of a row
// of one number (1 / n's rounding alone made 1 or -1 of 123 times 1e20).
__device__ __forceinline__ double mean_of(double sum, int64_t n, double inverse) {
    const double mean = sum * inverse;
    return __builtin_fma(__builtin_fma(-mean, static_cast<double>(n), sum), inverse, mean);
}

// `squares` over n numbers, of which `inverse` is 1 / n.
__device__ __forceinline__ Moments moments(int32_t kind, double mean, double squares, double inverse, float eps) {
    Moments m{0.0f, 0.0f, 1.0f, 1.0f};
    if (kind == SDHIP_ROW_NORM_NONE) return m;
    const float hi = static_cast<float>(mean);
    const double rest = mean - static_cast<double>(hi);
    const double r = inverse_root(__builtin_fma(squares, inverse, static_cast<double>(eps)));
    // A row without a spread, of whatever magnitude, stays: 0 times an infinity.
    const double power = r > 0x1p100 && r < __builtin_inf() ? 0x1p64 : r < 0x1p-100 ? 0x1p-64 : 1.0;
    m.power = static_cast<float>(power);
    m.scale = static_cast<float>(r > 0x1p100 ? r * 0x1p-64 : r < 0x1p-100 ? r * 0x1p64 : r);
    if (kind == SDHIP_ROW_NORM_LAYER) {
        m.hi = hi * m.power;
        m.lo = static_cast<float>(rest * power);
    }
    return m;
}

__device__ __forceinline__ float normed(float v, const Moments &m) {
    return __fmul_rn(__builtin_fmaf(v, m.power, -m.hi) - m.lo, m.scale);
}

// The sum of the wave's lanes, on all of them, the same bits: within rows of 16
// lanes by DPP, across them by swaps, which wait for no LDS as shuffles do
// (one row of 4096: 4.96 us by shuffles, so 4.59).
template <int CTRL>
__device__ __forceinline__ double moved(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t low = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(u), CTRL, 0xf, 0xf, true);
    const uint32_t high = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(u >> 32), CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, static_cast<uint64_t>(high) << 32 | low);
}

__device__ __forceinline__ double wave_sum(double v) {
    v += moved<0xb1>(v);   // lanes i ^ 1
    v += moved<0x4e>(v);   // i ^ 2
    v += moved<0x141>(v);  // 8 lanes mirrored
    v += moved<0x140>(v);  // 16 lanes mirrored
    const auto joined = [](const auto &low, const auto &high) {
        return __builtin_bit_cast(double, static_cast<uint64_t>(high[0]) << 32 | low[0]) +
               __builtin_bit_cast(double, static_cast<uint64_t>(high[1]) << 32 | low[1]);
    };
    uint64_t u = __builtin_bit_cast(uint64_t, v);
    uint32_t low = static_cast<uint32_t>(u), high = static_cast<uint32_t>(u >> 32);
    v = joined(__builtin_amdgcn_permlane16_swap(low, low, false, false), __builtin_amdgcn_permlane16_swap(high, high, false, false));
    u = __builtin_bit_cast(uint64_t, v);
    low = static_cast<uint32_t>(u);
    high = static_cast<uint32_t>(u >> 32);
    return joined(__builtin_amdgcn_permlane32_swap(low, low, false, false), __builtin_amdgcn_permlane32_swap(high, high, false, false));
}

}  // namespace sdhip
