// The norms after and before a transformer block with its gate and residual:
//     z = post(y),  s = residual_scale residual + branch_scale (gate z),  n = pre(s),
// a row's norm by its mean and the mean of its squares about it (LAYER), or
// about 0 (RMS), both summed in double: no square of a single-precision
// number passes it, and the mean is held in two single-precision parts.
//
// Bound by memory: each number of y and residual is read once and each of sum
// and out written once, the row in registers between its sums, T threads a
// row, up to 4 Q numbers each (norm_residual_rows_kernel); longer rows are
// read again for every sum (norm_residual_long_kernel).  2 x 4096 rows of 5120
// 119 us, 5.6 TB/s of their 671 MB; one row of 4096 4.65 us, of which a launch is 1.7
// and the rest two sums one after the other.

#include "host.h"
#include "profile.h"
#include "residual.h"

namespace sdhip {

namespace {

constexpr int kThreads = 256;

struct Place {
    uint32_t i1, i2, i3;
};

__device__ __forceinline__ int64_t row_at(const int64_t (&nb)[4], const Place &p) {
    return p.i1 * nb[1] + p.i2 * nb[2] + p.i3 * nb[3];
}

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
    const uint32_t row = static_cast<uint32_t>(a.first) + blockIdx.x;
    Place p;
    split_index(row, static_cast<uint32_t>(a.ne1), static_cast<uint32_t>(a.ne2), p.i1, p.i2, p.i3);
    const float *y = a.y != nullptr ? a.y + row_at(a.ynb, p) : nullptr;
    const float *r = a.residual + row_at(a.rnb, p);
    float *sum = a.sum != nullptr ? a.sum + row_at(a.snb, p) : nullptr;
    float *out = a.out != nullptr ? a.out + row_at(a.onb, p) : nullptr;
    const auto stats = [&](int32_t kind, float eps, auto value) {
        double mean = 0.0, squares = 0.0;
        if (kind == SDHIP_ROW_NORM_LAYER) {
            double s = 0.0;
            for (int64_t i = threadIdx.x; i < a.ne0; i += kThreads) s += static_cast<double>(value(i));
            mean = mean_of(block_sum(s, lds), a.ne0, a.inverse);
        }
        if (kind != SDHIP_ROW_NORM_NONE) {
            double s = 0.0;
            for (int64_t i = threadIdx.x; i < a.ne0; i += kThreads) {
                const double d = static_cast<double>(value(i)) - mean;
                s += d * d;
            }
            squares = block_sum(s, lds);
        }
        return moments(kind, mean, squares, a.inverse, eps);
    };
    const auto affine = [&](const RowNorm &w, float v, int64_t i) {
        if (w.weight.data != nullptr) {
            v = __fmul_rn(v, __fadd_rn(w.weight.data[row_at(w.weight.nb, p) + i * w.weight.nb[0]], w.offset));
        }
        if (w.bias.data != nullptr) v = __fadd_rn(v, w.bias.data[row_at(w.bias.nb, p) + i * w.bias.nb[0]]);
        return v;
    };
    Moments post{0.0f, 0.0f, 1.0f, 1.0f};
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

// T threads a row (T = 64: four rows a workgroup), each holding 4 Q numbers
// of it: Q quads T apart where rows lie at multiples of 16 bytes (QUADS), else
// 4 Q numbers T apart.
template <int T, int Q, bool QUADS>
__global__ __launch_bounds__(T == 64 ? 256 : T) void norm_residual_rows_kernel(ResidualArgs a) {
    __shared__ double lds[4][T / 64];  // a sum each: no sum waits for the one before to be read
    const int tid = T == 64 ? threadIdx.x & 63 : threadIdx.x;
    const uint32_t row = static_cast<uint32_t>(a.first) +
                         (T == 64 ? blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : blockIdx.x);
    if (row >= static_cast<uint32_t>(a.rows)) return;  // T = 64 only: its waves meet at no barrier
    Place p;
    split_index(row, static_cast<uint32_t>(a.ne1), static_cast<uint32_t>(a.ne2), p.i1, p.i2, p.i3);
    const int n = static_cast<int>(a.ne0);
    const auto at = [&](int u, int k) { return QUADS ? 4 * (tid + T * u) + k : tid + T * (4 * u + k); };
    const auto load = [&](const float *from, float (&v)[Q][4]) {
#pragma unroll
        for (int u = 0; u < Q; ++u) {
            if constexpr (QUADS) {
                float4v q = {0.0f, 0.0f, 0.0f, 0.0f};
                if (at(u, 0) < n) q = *reinterpret_cast<const float4v *>(from + at(u, 0));
#pragma unroll
                for (int k = 0; k < 4; ++k) v[u][k] = q[k];
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[u][k] = at(u, k) < n ? from[at(u, k)] : 0.0f;
            }
        }
    };
    const auto store = [&](float *to, const float (&v)[Q][4]) {
#pragma unroll
        for (int u = 0; u < Q; ++u) {
            if constexpr (QUADS) {
                if (at(u, 0) < n) *reinterpret_cast<float4v *>(to + at(u, 0)) = float4v{v[u][0], v[u][1], v[u][2], v[u][3]};
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (at(u, k) < n) to[at(u, k)] = v[u][k];
            }
        }
    };
    // An operand's numbers for the row: read as the rows are where it lies so,
    // else one number for all or each where it is.
    const auto operand = [&](const RowOperand &o, float (&v)[Q][4]) {
        const float *from = o.data + row_at(o.nb, p);
        if (o.nb[0] == 1 && (!QUADS || reinterpret_cast<uintptr_t>(from) % 16 == 0)) {
            load(from, v);
            return;
        }
#pragma unroll
        for (int u = 0; u < Q; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) v[u][k] = at(u, k) < n ? from[at(u, k) * o.nb[0]] : 0.0f;
    };
    int sums = 0;
    const auto total = [&](double v) {
        v = wave_sum(v);
        if constexpr (T > 64) {
            if ((tid & 63) == 0) lds[sums][tid >> 6] = v;
            __syncthreads();
            v = 0.0;
#pragma unroll
            for (int w = 0; w < T / 64; ++w) v += lds[sums][w];
            ++sums;
        }
        return v;
    };
    // Of numbers that are 0 past the row's.
    const auto stats = [&](int32_t kind, float eps, const float (&v)[Q][4]) {
        double mean = 0.0, squares = 0.0;
        if (kind == SDHIP_ROW_NORM_LAYER) {
            double s = 0.0;
#pragma unroll
            for (int u = 0; u < Q; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) s += static_cast<double>(v[u][k]);
            mean = mean_of(total(s), n, a.inverse);
        }
#pragma unroll
        for (int u = 0; u < Q; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const double d = at(u, k) < n ? static_cast<double>(v[u][k]) - mean : 0.0;
                squares = __builtin_fma(d, d, squares);
            }
        return moments(kind, mean, total(squares), a.inverse, eps);
    };
    const auto affine = [&](const RowNorm &w, float (&v)[Q][4]) {
        if (w.weight.data != nullptr) {
            float o[Q][4];
            operand(w.weight, o);
#pragma unroll
            for (int u = 0; u < Q; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[u][k] = __fmul_rn(v[u][k], __fadd_rn(o[u][k], w.offset));
        }
        if (w.bias.data != nullptr) {
            float o[Q][4];
            operand(w.bias, o);
#pragma unroll
            for (int u = 0; u < Q; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[u][k] = __fadd_rn(v[u][k], o[u][k]);
        }
    };
    float s[Q][4];
    if (a.y != nullptr) {
        float z[Q][4];
        load(a.y + row_at(a.ynb, p), z);
        load(a.residual + row_at(a.rnb, p), s);
        if (a.post.kind != SDHIP_ROW_NORM_NONE) {
            const Moments m = stats(a.post.kind, a.post.eps, z);
#pragma unroll
            for (int u = 0; u < Q; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) z[u][k] = normed(z[u][k], m);
            // Past the row's numbers the mean was taken from 0: they count in no
            // later mean (each number tested in the sums instead: 2 x 988 rows of 1280
            // 10.6 us, so 10.2).
            if (a.post.kind == SDHIP_ROW_NORM_LAYER && n < 4 * Q * T) {
#pragma unroll
                for (int u = 0; u < Q; ++u)
#pragma unroll
                    for (int k = 0; k < 4; ++k) z[u][k] = at(u, k) < n ? z[u][k] : 0.0f;
            }
        }
        affine(a.post, z);
        if (a.gate.data != nullptr) {
            float o[Q][4];
            operand(a.gate, o);
#pragma unroll
            for (int u = 0; u < Q; ++u)
#pragma unroll
                for (int k = 0; k < 4; ++k) z[u][k] = __fmul_rn(z[u][k], o[u][k]);
        }
#pragma unroll
        for (int u = 0; u < Q; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                s[u][k] = __fadd_rn(__fmul_rn(a.residual_scale, s[u][k]), __fmul_rn(a.branch_scale, z[u][k]));
    } else {
        load(a.residual + row_at(a.rnb, p), s);
#pragma unroll
        for (int u = 0; u < Q; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[u][k] = __fmul_rn(a.residual_scale, s[u][k]);
    }
    if (a.sum != nullptr) store(a.sum + row_at(a.snb, p), s);
    if (a.out == nullptr) return;
    if (a.pre.kind != SDHIP_ROW_NORM_NONE) {
        const Moments m = stats(a.pre.kind, a.pre.eps, s);
#pragma unroll
        for (int u = 0; u < Q; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[u][k] = normed(s[u][k], m);
    }
    affine(a.pre, s);
    store(a.out + row_at(a.onb, p), s);
}

// A launch holds 2^32 - 1 threads at most: 2^31 of them at a time, `threads` a row.
template <class Launch>
hipError_t by_rows(ResidualArgs a, int threads, Launch launch) {
    const int64_t most = (int64_t{1} << 31) / threads;
    for (; a.first < a.rows; a.first += most) {
        launch(a, a.rows - a.first < most ? a.rows - a.first : most);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <int T, int Q>
hipError_t launch_rows(const ResidualArgs &args, bool quads, hipStream_t stream) {
    return by_rows(args, T, [&](const ResidualArgs &a, int64_t rows) {
        const dim3 grid(static_cast<uint32_t>(T == 64 ? ceil_div(rows, 4) : rows)), block(T == 64 ? 256 : T);
        if (quads) {
            SDHIP_LAUNCH((norm_residual_rows_kernel<T, Q, true>), grid, block, 0, stream, a);
        } else {
            SDHIP_LAUNCH((norm_residual_rows_kernel<T, Q, false>), grid, block, 0, stream, a);
        }
    });
}

}  // namespace

hipError_t launch_norm_residual(const ResidualArgs &a, hipStream_t stream) {
    KernelScope scope("norm_residual", stream);
    const auto quads = [&](const float *p, const int64_t (&nb)[4]) {
        return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && nb[1] % 4 == 0 && nb[2] % 4 == 0 && nb[3] % 4 == 0);
    };
    const bool q = a.ne0 % 4 == 0 && quads(a.y, a.ynb) && quads(a.residual, a.rnb) && quads(a.sum, a.snb) && quads(a.out, a.onb);
    // As few threads a row as hold it in 16 or 20 numbers each, and of up to
    // 1280 numbers a wave alone where there are rows for every wave (2 x 988
    // rows of 1280: 10.6 us, by four waves 12.6; 512 rows 5.9 and 5.5; one row of
    // 4096 by four waves 5.0 us, by sixteen 5.6; 2 x 4096 rows of 5120 122 and 182),
    // in as few registers as hold it (2 x 4096 rows of 640 in 12 numbers a lane
    // 17.4 us, in 20 20.2).
    const bool many = a.rows >= 4 * static_cast<int64_t>(compute_units());
    if (a.ne0 <= 256) return launch_rows<64, 1>(a, q, stream);
    if (a.ne0 <= 512) return launch_rows<64, 2>(a, q, stream);
    if (many && a.ne0 <= 768) return launch_rows<64, 3>(a, q, stream);
    if (many && a.ne0 <= 1280) return launch_rows<64, 5>(a, q, stream);
    if (a.ne0 <= 1024) return launch_rows<256, 1>(a, q, stream);
    if (a.ne0 <= 2048) return launch_rows<256, 2>(a, q, stream);
    if (a.ne0 <= 4096) return launch_rows<256, 4>(a, q, stream);
    if (a.ne0 <= 5120) return launch_rows<256, 5>(a, q, stream);
    if (a.ne0 <= 8192) return launch_rows<512, 4>(a, q, stream);
    if (a.ne0 <= 16384) return launch_rows<1024, 4>(a, q, stream);
    return by_rows(a, kThreads, [&](const ResidualArgs &part, int64_t rows) {
        SDHIP_LAUNCH(norm_residual_long_kernel, dim3(static_cast<uint32_t>(rows)), dim3(kThreads), 0, stream, part);
    });
}

}  // namespace sdhip
