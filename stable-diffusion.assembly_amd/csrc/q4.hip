// MUL_MAT of weights in ggml's 4-bit blocks (Q4_0, Q4_1): each block of 32
// weights along K is a half-precision scale d, with Q4_1 a half-precision
// least value m, and 16 bytes, byte j holding number j in its low four bits
// and number 16 + j in its high ones.  Both types are one:
//     w = d (q - 8) + c,   c = 0 (Q4_0) or m + 8 d (Q4_1),
// so that a block's part of an output is d sum((q - 8) x) + c sum(x), q - 8 a
// whole number of -8 .. 7.

#include <hip/hip_fp16.h>

#include "host.h"
#include "profile.h"
#include "q4.h"

namespace sdhip {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float half_at(const uint8_t *p) {
    _Float16 h;
    __builtin_memcpy(&h, p, 2);
    return static_cast<float>(h);
}

// An output a wave: its lanes take blocks 64 apart.
template <bool LEAST, bool GATED>
__global__ __launch_bounds__(kThreads) void q4_simple_kernel(Q4Args a) {
    constexpr int kSize = LEAST ? 20 : 18;
    const int64_t columns = GATED ? a.half : a.N;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
    if (item >= columns * a.M) return;
    const int lane = threadIdx.x & 63;
    const int64_t m = item / columns, n = item - m * columns;
    const float *x = a.x + m * a.ldx;
    float sums[GATED ? 2 : 1];
#pragma unroll
    for (int p = 0; p < (GATED ? 2 : 1); ++p) {
        const uint8_t *row = a.w + (n + p * a.half) * a.row_bytes;
        float s = 0.0f;
        for (int64_t b = lane; b < a.K / kBlock; b += 64) {
            const uint8_t *block = row + b * kSize;
            const float d = half_at(block);
            const float c = LEAST ? __builtin_fmaf(8.0f, d, half_at(block + 2)) : 0.0f;
            float q = 0.0f, t = 0.0f;
            for (int j = 0; j < 16; ++j) {
                const int byte = block[kSize - 16 + j];
                const float x0 = x[b * kBlock + j], x1 = x[b * kBlock + 16 + j];
                q = __builtin_fmaf(static_cast<float>((byte & 15) - 8), x0, q);
                q = __builtin_fmaf(static_cast<float>((byte >> 4) - 8), x1, q);
                t += x0 + x1;
            }
            s = __builtin_fmaf(d, q, s);
            if (LEAST) s = __builtin_fmaf(c, t, s);
        }
        for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
        sums[p] = s;
    }
    if (lane != 0) return;
    uint32_t i1, i2, i3;
    split_index(static_cast<uint32_t>(m), static_cast<uint32_t>(a.ne1), static_cast<uint32_t>(a.ne2), i1, i2, i3);
    if (a.from_redirect) sums[0] = a.y[m * a.ldy + n] + sums[0];
    apply_chain_block(a.chain, sums, [&](int s, int p) {
        const DevStep &st = a.chain.steps[s];
        return (n + p * a.half) * st.nb[0] + i1 * st.nb[1] + i2 * st.nb[2] + i3 * st.nb[3];
    });
    a.y[m * a.ldy + n] = GATED ? sums[0] * gelu(sums[GATED ? 1 : 0]) : sums[0];
}

}  // namespace

hipError_t launch_q4_mul_mat(const Q4Args &a, hipStream_t stream) {
    KernelScope scope(a.half ? "q4.gated" : "q4", stream);
    const dim3 grid(static_cast<uint32_t>(ceil_div((a.half ? a.half : a.N) * a.M, kThreads / 64)));
    if (a.half) {
        if (a.least) {
            SDHIP_LAUNCH((q4_simple_kernel<true, true>), grid, dim3(kThreads), 0, stream, a);
        } else {
            SDHIP_LAUNCH((q4_simple_kernel<false, true>), grid, dim3(kThreads), 0, stream, a);
        }
    } else if (a.least) {
        SDHIP_LAUNCH((q4_simple_kernel<true, false>), grid, dim3(kThreads), 0, stream, a);
    } else {
        SDHIP_LAUNCH((q4_simple_kernel<false, false>), grid, dim3(kThreads), 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace sdhip
