// The outputs of a workgroup whose waves hold sums over parts of K (q4.hip,
// f8.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device.h"

namespace sdhip {

// The outputs of a workgroup of `threads` from its splits' sums in LDS, `step`
// apart, `count` outputs, with GATED the second half's behind them: their sums
// in the splits' order, times what `place` gives with an output's row (M or
// more: none) and column; the redirect's number first, the chain, the gated
// GELU.  E of a thread's at a time, so that their loads go out together.
template <bool GATED, int E, class Args, class Place>
__device__ __forceinline__ void write_outputs(const Args &a, const float *sums, int splits, int step, int count, int tid,
                                              int columns, Place place, int threads) {
    constexpr int kHalves = GATED ? 2 : 1, kMost = 8;  // the most splits there are
#pragma unroll 1
    for (int first = tid; first < count; first += E * threads) {
        int64_t m[E];
        int n[E];
        bool real[E];
        float v[kHalves * E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int at = first + threads * e < count ? first + threads * e : first;
            const float back = place(at, m[e], n[e]);
            real[e] = first + threads * e < count && m[e] < a.M && n[e] < columns;
            m[e] = m[e] < a.M ? m[e] : a.M - 1;
            n[e] = n[e] < columns ? n[e] : columns - 1;
#pragma unroll
            for (int p = 0; p < kHalves; ++p) {
                float s[kMost];
#pragma unroll
                for (int k = 0; k < kMost; ++k) s[k] = sums[(k < splits ? k : 0) * step + p * count + at];
                float total = s[0];
#pragma unroll
                for (int k = 1; k < kMost; ++k) total = k < splits ? total + s[k] : total;
                v[kHalves * e + p] = total * back;
            }
        }
        if (!GATED && a.from_redirect) {
#pragma unroll
            for (int e = 0; e < E; ++e) v[kHalves * e] = a.y[m[e] * a.ldy + n[e]] + v[kHalves * e];
        }
        apply_chain_block(a.chain, v, [&](int s, int i) {
            const DevStep &st = a.chain.steps[s];
            const int64_t at = (n[i / kHalves] + (i % kHalves) * static_cast<int64_t>(columns)) * st.nb[0];
            const int64_t row = m[i / kHalves];
            if (st.flat123) return at + row * st.nb[1];
            uint32_t i1, i2, i3;
            split_index(static_cast<uint32_t>(row), static_cast<uint32_t>(a.ne1), static_cast<uint32_t>(a.ne2), i1, i2, i3);
            return at + i1 * st.nb[1] + i2 * st.nb[2] + i3 * st.nb[3];
        });
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (real[e]) a.y[m[e] * a.ldy + n[e]] = GATED ? v[kHalves * e] * gelu(v[kHalves * e + kHalves - 1]) : v[kHalves * e];
        }
    }
}

}  // namespace sdhip
