// Rotary positions of several axes after the norm of each head's numbers: the
// pair (u, v) of numbers that an axis turns by an angle t becomes
//     (u cos t - v sin t, u sin t + v cos t),   t = position base^(-2 j / dims).
// An angle is taken in double and brought to a quarter of a turn before its sine
// and cosine in single precision, so that one of 10^7 turns keeps its 2^-24.
//
// Bound by memory, each number read and written once.  A wave takes a token and a
// part of its heads: the token's sines and cosines are computed once, a pair a
// lane, and shared through LDS by the heads, a row of which takes 8, 16 or 64 lanes,
// each with 8 numbers of it (or 16): those of four pairs.  64 x 64 tokens of 48 heads of
// 128 with a norm take 34 us, 5.9 TB/s; 21 x 30 x 52 of 12 heads to FP16 68, 4.4; one
// token of 32 heads 3.9, a launch and the position's, the sine's and x's latencies.

#include <type_traits>

#include "host.h"
#include "profile.h"
#include "rope.h"

namespace sdhip {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// cos and sin of `turns` half turns: of what is left of them by the nearest quarter
// of a turn, 45 degrees at most, by Taylor's series to x^9 and x^10 (off by 2e-9 of
// themselves), in the quarter's place.  The quarters are counted in the last bits of
// a sum with 1.5 x 2^52.
__device__ __forceinline__ float2 turn(double turns) {
    const double magic = 6755399441055744.0, sum = __builtin_fma(2.0, turns, magic), q = sum - magic;
    const float x = static_cast<float>(3.14159265358979323846 * __builtin_fma(-0.5, q, turns)), x2 = x * x;
    float s = __builtin_fmaf(x2, 2.7557319e-6f, -1.9841270e-4f);
    s = __builtin_fmaf(s, x2, 8.3333333e-3f);
    s = __builtin_fmaf(s, x2, -1.6666667e-1f);
    s = __builtin_fmaf(x * x2, s, x);
    float c = __builtin_fmaf(x2, -2.7557319e-7f, 2.4801587e-5f);
    c = __builtin_fmaf(c, x2, -1.3888889e-3f);
    c = __builtin_fmaf(c, x2, 4.1666667e-2f);
    c = __builtin_fmaf(c, x2, -0.5f);
    c = __builtin_fmaf(c, x2, 1.0f);
    const uint32_t k = static_cast<uint32_t>(__builtin_bit_cast(uint64_t, sum));
    const float2 t = k & 1 ? make_float2(-s, c) : make_float2(c, s);
    return k & 2 ? make_float2(-t.x, -t.y) : t;
}

// The sum of a row's LPR lanes, on all of them.
template <int LPR>
__device__ __forceinline__ double row_sum(double v) {
    if constexpr (LPR == 64) return wave_sum(v);
    v += moved<0xb1>(v);   // lanes i ^ 1
    v += moved<0x4e>(v);   // i ^ 2
    v += moved<0x141>(v);  // 8 lanes mirrored
    if constexpr (LPR == 16) v += moved<0x140>(v);  // 16 lanes mirrored
    return v;
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
    const auto add = [](float v, auto control) {
        return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(control)::value, 0xf, 0xf, true));
    };
    v = add(v, std::integral_constant<int, 0xb1>{});
    v = add(v, std::integral_constant<int, 0x4e>{});
    v = add(v, std::integral_constant<int, 0x141>{});
    if constexpr (LPR >= 16) v = add(v, std::integral_constant<int, 0x140>{});
    if constexpr (LPR == 64) {
        uint32_t a = __builtin_bit_cast(uint32_t, v), b = a;
        swap16(a, b);
        v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
        a = b = __builtin_bit_cast(uint32_t, v);
        swap32(a, b);
        v = __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
    }
    return v;
}

// LPR lanes a row, SLOTS groups of four pairs each; QUADS where every four
// numbers that a lane reads or writes at once lie at a multiple of their size; FEW
// where a token's heads are half of a wave's rows or fewer: it takes rows of as many
// tokens as there is room for, and each lane computes its own pairs' sines and cosines
// (50688 tokens of one head of 40 32 us by a token a wave, so 10.6; 4096 of two of 128 6.5
// and 5.7, but 2048 5.1 and 5.3: where waves are as many as tokens four turns a lane take
// longer than one).
template <int LPR, int SLOTS, bool ADJACENT, bool QUADS, bool FEW>
__global__ __launch_bounds__(kThreads, SLOTS == 1 ? 4 : 1) void rope_kernel(RopeArgs a) {
    __shared__ float2 shared[FEW ? 1 : kWaves][FEW ? 1 : 64 * (LPR * SLOTS <= 16 ? 1 : LPR * SLOTS <= 32 ? 2 : 4)];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int pairs = a.turned / 2;
    float2 *turns = shared[FEW ? 0 : wave];
    const int sub = lane % LPR;
    // The frequencies, in half turns, of the pairs that this lane computes: each 64th of
    // a token's, or its own.
    constexpr int kMine = FEW ? 4 * SLOTS : LPR * SLOTS <= 16 ? 1 : LPR * SLOTS <= 32 ? 2 : 4;
    double rate[kMine];
    int axis[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int p = FEW ? 4 * (sub + LPR * (i / 4)) + i % 4 : lane + 64 * i;
        axis[i] = 0;
#pragma unroll
        for (int j = 1; j < SDHIP_MAX_AXES; ++j)
            if (j < a.count && p >= a.first[j]) axis[i] = j;
        rate[i] = FEW || 64 * i < pairs ? exp2(a.rate[axis[i]] * (p - a.from[axis[i]])) * 0.31830988618379067154 : 0.0;
    }
    // This lane's pairs: the place of each one's numbers, d or more where there is none.
    const int front = ADJACENT ? 0 : (pairs + 3) / 4;  // groups of halves' pairs, before those that are not turned
    int at[SLOTS][4][2];
    bool turned[SLOTS][4];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int group = sub + LPR * s;
            if (ADJACENT) {
                const int p = 4 * group + c;
                at[s][c][0] = 2 * p;
                at[s][c][1] = 2 * p + 1;
                turned[s][c] = p < pairs;
            } else if (group < front) {
                const int p = 4 * group + c;
                at[s][c][0] = p < pairs ? p : a.d;
                at[s][c][1] = p < pairs ? p + pairs : a.d;
                turned[s][c] = p < pairs;
            } else {
                const int i = a.turned + 8 * (group - front) + c;
                at[s][c][0] = i;
                at[s][c][1] = i + 4;
                turned[s][c] = false;
            }
        }
    // With QUADS the numbers of a group are two runs of four: an ADJACENT one's
    // pairs are within them, a HALVES one's across.
    const auto load = [&](const float *row, bool quads, int64_t step, float (&v)[SLOTS][4][2]) {
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            if (QUADS && quads) {
                float4v q[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int i = ADJACENT ? at[s][2 * h][0] : at[s][0][h];
                    q[h] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
                    if (i < a.d) q[h] = *reinterpret_cast<const float4v *>(row + i);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int h = 0; h < 2; ++h) v[s][c][h] = ADJACENT ? q[c / 2][2 * (c % 2) + h] : q[h][c];
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int h = 0; h < 2; ++h) v[s][c][h] = at[s][c][h] < a.d ? row[at[s][c][h] * step] : 0.0f;
            }
        }
    };
    const auto store = [&](auto *row, const float (&v)[SLOTS][4][2]) {
        typedef std::conditional_t<sizeof(*row) == 2, half4, float4v> Four;
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            if constexpr (QUADS) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int i = ADJACENT ? at[s][2 * h][0] : at[s][0][h];
                    Four q;
#pragma unroll
                    for (int c = 0; c < 4; ++c) q[c] = ADJACENT ? v[s][2 * h + c / 2][c % 2] : v[s][c][h];
                    if (i < a.d) *reinterpret_cast<Four *>(row + i) = q;
                }
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (at[s][c][h] < a.d) row[at[s][c][h]] = static_cast<std::remove_reference_t<decltype(*row)>>(v[s][c][h]);
            }
        }
    };
    const auto quads_of = [&](const RowOperand &o) {
        return QUADS && o.nb[0] == 1 && reinterpret_cast<uintptr_t>(o.data) % 16 == 0 && o.nb[1] % 4 == 0 && o.nb[2] % 4 == 0 &&
               o.nb[3] % 4 == 0;
    };
    const bool weight_quads = quads_of(a.norm.weight), bias_quads = quads_of(a.norm.bias);
    constexpr int kRows = 64 / LPR;  // heads of a wave at a time
    // A row's norm and turns; a row's lanes together.
    const auto row = [&](const float *x, const float *weight, const float *bias, int64_t to, const float2 (&by)[SLOTS][4]) {
        float v[SLOTS][4][2];
        load(x, true, 1, v);
        if (a.norm.kind != SDHIP_ROW_NORM_NONE) {
            float sum = 0.0f;
            if (a.norm.kind == SDHIP_ROW_NORM_RMS) {
#pragma unroll
                for (int s = 0; s < SLOTS; ++s)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int k = 0; k < 2; ++k) sum = __builtin_fmaf(v[s][c][k], v[s][c][k], sum);
                sum = row_sum<LPR>(sum);
            }
            if (a.norm.kind == SDHIP_ROW_NORM_RMS && sum > 0x1p-60f && sum < 0x1p100f) {
                const float scale = __builtin_amdgcn_rsqf(__builtin_fmaf(sum, static_cast<float>(a.inverse), a.norm.eps));
#pragma unroll
                for (int s = 0; s < SLOTS; ++s)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int k = 0; k < 2; ++k) v[s][c][k] *= scale;
            } else {
                // In double: means, and squares near single precision's limits.
                double mean = 0.0, squares = 0.0;
                if (a.norm.kind == SDHIP_ROW_NORM_LAYER) {
#pragma unroll
                    for (int s = 0; s < SLOTS; ++s)
#pragma unroll
                        for (int c = 0; c < 4; ++c) mean += static_cast<double>(v[s][c][0]) + static_cast<double>(v[s][c][1]);
                    mean = mean_of(row_sum<LPR>(mean), a.d, a.inverse);
                }
#pragma unroll
                for (int s = 0; s < SLOTS; ++s)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const double d = at[s][c][k] < a.d ? static_cast<double>(v[s][c][k]) - mean : 0.0;
                            squares = __builtin_fma(d, d, squares);
                        }
                const Moments m = moments(a.norm.kind, mean, row_sum<LPR>(squares), a.inverse, a.norm.eps);
#pragma unroll
                for (int s = 0; s < SLOTS; ++s)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int k = 0; k < 2; ++k) v[s][c][k] = normed(v[s][c][k], m);
            }
        }
        if (weight != nullptr) {
            float w[SLOTS][4][2];
            load(weight, weight_quads, a.norm.weight.nb[0], w);
#pragma unroll
            for (int s = 0; s < SLOTS; ++s)
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int k = 0; k < 2; ++k) v[s][c][k] = __fmul_rn(v[s][c][k], __fadd_rn(w[s][c][k], a.norm.offset));
        }
        if (bias != nullptr) {
            float w[SLOTS][4][2];
            load(bias, bias_quads, a.norm.bias.nb[0], w);
#pragma unroll
            for (int s = 0; s < SLOTS; ++s)
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int k = 0; k < 2; ++k) v[s][c][k] = __fadd_rn(v[s][c][k], w[s][c][k]);
        }
#pragma unroll
        for (int s = 0; s < SLOTS; ++s)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float one = v[s][c][0], two = v[s][c][1], cosine = by[s][c].x, sine = by[s][c].y;
                const float u = __builtin_fmaf(-two, sine, one * cosine), w = __builtin_fmaf(one, sine, two * cosine);
                // Not turned: as they are, whatever the other of the two is.
                v[s][c][0] = turned[s][c] ? u : one;
                v[s][c][1] = turned[s][c] ? w : two;
            }
        if (a.half) {
            store(static_cast<_Float16 *>(a.y) + to, v);
        } else {
            store(static_cast<float *>(a.y) + to, v);
        }
    };
    const int mine = lane / LPR;
    const int64_t tokens = a.tokens * a.batch, step = static_cast<int64_t>(gridDim.x) * kWaves;
    if constexpr (FEW) {
        const int64_t items = (tokens * a.heads + kRows - 1) / kRows;
        for (int64_t item = static_cast<int64_t>(blockIdx.x) * kWaves + wave; item < items; item += step) {
            const int64_t first = item * kRows / a.heads;  // the token of the wave's first row
            const int ahead = static_cast<int>(item * kRows - first * a.heads) + mine, skip = ahead / a.heads, h = ahead - skip * a.heads;
            if (first + skip >= tokens) continue;
            int64_t i3 = first / a.tokens, i1 = first - i3 * a.tokens + skip;
            while (i1 >= a.tokens) {
                i1 -= a.tokens;
                ++i3;
            }
            const float *positions = a.positions + i1 * a.pnb1 + i3 * a.pnb3;
            float2 by[SLOTS][4];
#pragma unroll
            for (int s = 0; s < SLOTS; ++s)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    by[s][c] = turned[s][c] ? turn(static_cast<double>(positions[axis[4 * s + c]]) * rate[4 * s + c]) : make_float2(1.0f, 0.0f);
            const auto of = [&](const RowOperand &o) { return o.data != nullptr ? o.data + i1 * o.nb[1] + i3 * o.nb[3] + h * o.nb[2] : nullptr; };
            row(a.x + i1 * a.xnb[1] + i3 * a.xnb[3] + h * a.xnb[2], of(a.norm.weight), of(a.norm.bias),
                i1 * a.ynb[1] + i3 * a.ynb[3] + h * a.ynb[2], by);
        }
        return;
    }
    const int share = (a.heads + a.parts - 1) / a.parts;
    // How far a lane's row lies from the wave's first.
    const int64_t x_lane = lane / LPR * a.xnb[2], y_lane = lane / LPR * a.ynb[2];
    const int64_t w_lane = lane / LPR * a.norm.weight.nb[2], b_lane = lane / LPR * a.norm.bias.nb[2];
    const int64_t items = tokens * a.parts;
    for (int64_t item = static_cast<int64_t>(blockIdx.x) * kWaves + wave; item < items; item += step) {
        const int64_t token = item / a.parts;
        const int part = static_cast<int>(item - token * a.parts);
        const int64_t i3 = token / a.tokens, i1 = token - i3 * a.tokens;
        const float *positions = a.positions + i1 * a.pnb1 + i3 * a.pnb3;
        // The turns of the token before are read.
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < kMine; ++i)
            if (64 * i < pairs && lane + 64 * i < pairs) turns[lane + 64 * i] = turn(static_cast<double>(positions[axis[i]]) * rate[i]);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        float2 by[SLOTS][4];
#pragma unroll
        for (int s = 0; s < SLOTS; ++s)
#pragma unroll
            for (int c = 0; c < 4; ++c) by[s][c] = turned[s][c] ? turns[4 * (sub + LPR * s) + c] : make_float2(1.0f, 0.0f);
        const int h0 = part * share, h1 = h0 + share < a.heads ? h0 + share : a.heads;
        const float *x = a.x + i1 * a.xnb[1] + i3 * a.xnb[3] + h0 * a.xnb[2] + x_lane;
        int64_t to = i1 * a.ynb[1] + i3 * a.ynb[3] + h0 * a.ynb[2] + y_lane;
        const float *weight = a.norm.weight.data, *bias = a.norm.bias.data;
        if (weight != nullptr) weight += i1 * a.norm.weight.nb[1] + i3 * a.norm.weight.nb[3] + h0 * a.norm.weight.nb[2] + w_lane;
        if (bias != nullptr) bias += i1 * a.norm.bias.nb[1] + i3 * a.norm.bias.nb[3] + h0 * a.norm.bias.nb[2] + b_lane;
        for (int h = h0; h < h1; h += kRows) {
            if (h + mine >= h1) continue;  // a row's lanes together
            row(x, weight, bias, to, by);
            x += kRows * a.xnb[2];
            if (weight != nullptr) weight += kRows * a.norm.weight.nb[2];
            if (bias != nullptr) bias += kRows * a.norm.bias.nb[2];
            to += kRows * a.ynb[2];
        }
    }
}

template <int LPR, int SLOTS, bool FEW>
hipError_t launch(const RopeArgs &a, bool quads, dim3 grid, hipStream_t stream) {
    const dim3 block(kThreads);
    if (a.order == SDHIP_ROPE_ADJACENT) {
        if (quads) {
            SDHIP_LAUNCH((rope_kernel<LPR, SLOTS, true, true, FEW>), grid, block, 0, stream, a);
        } else {
            SDHIP_LAUNCH((rope_kernel<LPR, SLOTS, true, false, FEW>), grid, block, 0, stream, a);
        }
    } else if (quads) {
        SDHIP_LAUNCH((rope_kernel<LPR, SLOTS, false, true, FEW>), grid, block, 0, stream, a);
    } else {
        SDHIP_LAUNCH((rope_kernel<LPR, SLOTS, false, false, FEW>), grid, block, 0, stream, a);
    }
    return hipGetLastError();
}

template <int LPR, int SLOTS>
hipError_t launch(RopeArgs a, bool quads, hipStream_t stream) {
    constexpr int64_t kRows = 64 / LPR;
    const int64_t waves = 16 * static_cast<int64_t>(compute_units()), tokens = a.tokens * a.batch;
    const auto grid = [&](int64_t items) { return dim3(static_cast<uint32_t>(ceil_div(items < 2 * waves ? items : 2 * waves, kWaves))); };
    if constexpr (LPR < 64 && SLOTS == 1) {
        if (2 * a.heads <= kRows && tokens >= waves) return launch<LPR, SLOTS, true>(a, quads, grid(ceil_div(tokens * a.heads, kRows)), stream);
    }
    // Parts of a token's heads until every wave of the device has one, 16 a CU.
    const int64_t most = ceil_div(a.heads, kRows);
    a.parts = static_cast<int32_t>(tokens * most <= waves ? most : tokens >= waves ? 1 : ceil_div(waves, tokens));
    return launch<LPR, SLOTS, false>(a, quads, grid(tokens * a.parts), stream);
}

}  // namespace

hipError_t launch_rope(RopeArgs a, hipStream_t stream) {
    KernelScope scope("rope", stream);
    const auto strides = [](const int64_t (&nb)[4]) { return nb[1] % 4 == 0 && nb[2] % 4 == 0 && nb[3] % 4 == 0; };
    const bool quads = a.d % 4 == 0 && (a.order == SDHIP_ROPE_ADJACENT || a.turned % 8 == 0) && strides(a.xnb) && strides(a.ynb) &&
                       reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && reinterpret_cast<uintptr_t>(a.y) % (a.half ? 8 : 16) == 0;
    // Groups of four pairs of a row; a HALVES row's numbers that are not turned
    // are groups of their own.
    const int groups = static_cast<int>(a.order == SDHIP_ROPE_ADJACENT ? ceil_div(a.d, 8)
                                                                       : ceil_div(a.turned, 8) + ceil_div(a.d - a.turned, 8));
    if (groups <= 8) return launch<8, 1>(a, quads, stream);
    if (groups <= 16) return launch<16, 1>(a, quads, stream);
    if (groups <= 32) return launch<16, 2>(a, quads, stream);
    return launch<64, 2>(a, quads, stream);
}

}  // namespace sdhip
