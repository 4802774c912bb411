// MUL_MAT of 8-bit floating-point weights (E4M3), a single-precision scale for
// each block of 128 x 128 of them.
//
//     y[m][n] = sum over blocks b of s[n / 128][b] 2^e[m][b] sum over k in b of w[n][k] q[m][k]
//
// with row m's numbers of block b held as q 2^e: e the least whole number that
// brings their greatest magnitude to 448 or less, q E4M3 to nearest, ties to even.
// A power of two costs a floating-point format nothing (its numbers are as close
// at any magnitude but the least) and makes x 2^-e exact, so that q has one rounding
// and one value whoever computes it.
//
// The products are FP16's: the MFMA of 8 bits, of twice their rate, adds eight
// products at a time and keeps of each what is not below 2^-13 of the greatest
// (measured: 1e-4 of the products' magnitudes lost where they span 2^14, 6e-6 where
// 2^4), which is no sum in single precision; FP16's sums lose 2^-22 of them.  All of
// E4M3 is in FP16, two numbers by one v_cvt_scalef32_pk_f16_fp8.
//
// The weights are the MFMA's rows and x's rows its columns, so that a lane's sums
// are of one row of x: 2^e is the lane's own, s the same for all of 32 columns of the
// output, and a block's sums go to the outputs' by one multiplication a lane and an
// addition each.

#include <algorithm>

#include "f8.h"
#include "host.h"
#include "outputs.h"
#include "profile.h"

namespace sdhip {

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));

constexpr int kBlock = static_cast<int>(kF8Block);
constexpr int kLeast = -101 + 127;  // e's least, biased as an exponent's bits
constexpr uint32_t kNans = 0x7f7f7f7fu;  // four NaN of E4M3
constexpr uint32_t kInfinity = 0x7f800000u;

// ------------------------------------------------------------------ numbers

// e's bits, biased by 127, for a greatest magnitude of these bits: 448 is 1.75 x
// 2^8.  Those of an infinity or NaN are not used.
__device__ __forceinline__ uint32_t power_of(uint32_t greatest) {
    const int e = static_cast<int>((greatest + 0x1fffffu) >> 23) - 8;
    return static_cast<uint32_t>(e > kLeast ? e : kLeast);
}

// 2^e and 2^-e, e at most 120.
__device__ __forceinline__ float up(uint32_t e) { return __builtin_bit_cast(float, e << 23); }
__device__ __forceinline__ float down(uint32_t e) { return __builtin_bit_cast(float, (254 - e) << 23); }

__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t greater(uint32_t a, uint32_t b) { return a > b ? a : b; }

// Eight numbers of E4M3 as FP16.
__device__ __forceinline__ half8 widen(int low, int high) {
    const half2v a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(low, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(low, 1.0f, true);
    const half2v c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(high, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(high, 1.0f, true);
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Four numbers times `scale` as E4M3, those of a group with an infinity or NaN as
// NaN.
__device__ __forceinline__ int four(const float4v &v, float scale, bool finite) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * scale, v[1] * scale, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * scale, v[3] * scale, r, true);
    return finite ? r : static_cast<int>(kNans);
}

// Four of a row's K numbers from k on, 0 past its end.
__device__ __forceinline__ float4v load_x(const float *row, int64_t k, int64_t K) {
    if (k + 4 <= K) return load4(row + k);
    float4v v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (k + i < K) v[i] = row[k + i];
    return v;
}

// 16 of a row's K weights from k on, 0 past its end: of what follows a row
// nothing is read, since it may be no memory or hold NaN.
__device__ __forceinline__ int4v load_w(const uint8_t *row, int64_t k, int64_t K) {
    int4v v = {0, 0, 0, 0};
    if (k + 16 <= K) {
        __builtin_memcpy(&v, row + k, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 15; ++i)
            if (k + i < K) v[i / 4] |= static_cast<int>(row[k + i]) << (8 * (i % 4));
    }
    return v;
}

// ------------------------------------------------------------------ the work buffer

// x's q in FP16 as rows of whole blocks, zeros past K, and its 2^e, [block][row];
// the weights as rows of whole blocks, zeros past K, where the tiles need them so.
struct F8Work {
    _Float16 *q;
    float *powers;
    uint8_t *w;
    int64_t ld;    // K rounded up to whole blocks
    int64_t rows;  // of `powers`: M rounded up
    size_t bytes;
};

F8Work work_of(int64_t M, int64_t N, int64_t K, bool weights, void *work) {
    F8Work w{};
    w.ld = round_up(K, kF8Block);
    w.rows = round_up(M, 128);
    char *p = static_cast<char *>(work);
    size_t at = 0;
    const auto take = [&](int64_t bytes) {
        const size_t from = at;
        at += static_cast<size_t>(round_up(bytes, 256));
        return p != nullptr ? p + from : nullptr;
    };
    w.q = reinterpret_cast<_Float16 *>(take(2 * M * w.ld));
    w.powers = reinterpret_cast<float *>(take(4 * w.rows * (w.ld / kF8Block)));
    if (weights) w.w = reinterpret_cast<uint8_t *>(take(N * w.ld));
    w.bytes = at;
    return w;
}

constexpr int kOperandThreads = 256;

struct OperandsArgs {
    F8Args a;
    F8Work w;
    uint32_t blocks, groups;  // of K; of all of x
    uint32_t x_grid;          // the workgroups that lay out x
};

// A group of x by 16 lanes, 8 numbers each; behind them the weights' rows, 16
// numbers a lane.
__global__ __launch_bounds__(kOperandThreads) void f8_operands_kernel(OperandsArgs o) {
    const F8Args &a = o.a;
    if (blockIdx.x >= o.x_grid) {
        const int64_t pieces = o.w.ld / 16;
        const int64_t i = static_cast<int64_t>(blockIdx.x - o.x_grid) * kOperandThreads + threadIdx.x;
        const int64_t n = i / pieces, k = (i - n * pieces) * 16;
        if (n < a.N) *reinterpret_cast<int4v *>(o.w.w + n * o.w.ld + k) = load_w(a.w + n * a.row_bytes, k, a.K);
        return;
    }
    const uint32_t g = blockIdx.x * (kOperandThreads / 16) + threadIdx.x / 16;
    if (g >= o.groups) return;  // the 16 lanes of a group together
    const uint32_t m = g / o.blocks, b = g - m * o.blocks;
    const int64_t k = static_cast<int64_t>(b) * kBlock + 8 * (threadIdx.x & 15);
    const float *row = a.x + m * a.ldx;
    float4v v[2];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        v[i] = load_x(row, k + 4 * i, a.K);
#pragma unroll
        for (int j = 0; j < 4; ++j) top = greater(top, magnitude(v[i][j]));
    }
    top = greater(top, __builtin_amdgcn_update_dpp(0, top, 0xb1, 0xf, 0xf, true));   // lanes i ^ 1
    top = greater(top, __builtin_amdgcn_update_dpp(0, top, 0x4e, 0xf, 0xf, true));   // i ^ 2
    top = greater(top, __builtin_amdgcn_update_dpp(0, top, 0x141, 0xf, 0xf, true));  // 8 lanes mirrored
    top = greater(top, __builtin_amdgcn_update_dpp(0, top, 0x140, 0xf, 0xf, true));  // 16 lanes mirrored
    const uint32_t e = power_of(top);
    const float scale = down(e);
    const bool finite = top < kInfinity;
    *reinterpret_cast<half8 *>(o.w.q + m * o.w.ld + k) = widen(four(v[0], scale, finite), four(v[1], scale, finite));
    if ((threadIdx.x & 15) == 0) o.w.powers[b * o.w.rows + m] = finite ? up(e) : 1.0f;
}

// ------------------------------------------------------------------ few rows

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;

struct RowsArgs {
    F8Args a;
    F8Work w;
    int32_t splits;  // of K, a wave each; the other waves take further columns
    uint32_t column_blocks;
};

// A workgroup takes 16 RM rows of x and kWaves / splits tiles of 16 columns, a
// wave a tile (with GATED its columns of both halves) and every splits-th block of
// K; its operands come straight from memory into registers, and the splits' sums
// are joined in LDS.  x comes from the work buffer (LAID) or, for up to 16 rows, as
// it is: a lane holds the 32 numbers of a row's group that the MFMA wants of it, and
// four lanes have the group's greatest between them.
template <bool GATED, bool LAID, int RM>
__global__ __launch_bounds__(kThreads) void f8_rows_kernel(RowsArgs f) {
    const F8Args &a = f.a;
    constexpr int RN = GATED ? 2 : 1;
    extern __shared__ __attribute__((aligned(16))) float sums[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, group = lane >> 4;
    const int S = f.splits, P = kWaves / S;
    const int split = wave % S, tile = wave / S;
    const uint32_t row_block = blockIdx.x / f.column_blocks;
    const int64_t m0 = static_cast<int64_t>(row_block) * (16 * RM);
    const int columns = static_cast<int>(GATED ? a.half : a.N);
    const int n0 = static_cast<int>(blockIdx.x - row_block * f.column_blocks) * (16 * P);
    const int blocks = static_cast<int>((a.K + kBlock - 1) / kBlock);
    const int n = n0 + 16 * tile;
    const uint8_t *w[RN];
    const float *scales[RN][2];  // of the lane's first output and of its last, which lie in two blocks at most
    int across[RN];              // the outputs of the lane in the first one's block
#pragma unroll
    for (int j = 0; j < RN; ++j) {
        const int64_t from = j ? columns : 0;
        w[j] = a.w + (from + (n + col < columns ? n + col : columns - 1)) * a.row_bytes;
        const int64_t low = from + (n + 4 * group < columns ? n + 4 * group : columns - 1);
        const int64_t high = low + 3 < a.N ? low + 3 : a.N - 1;
        scales[j][0] = a.scales + low / kBlock * a.ld_scales;
        scales[j][1] = a.scales + high / kBlock * a.ld_scales;
        across[j] = kBlock - static_cast<int>(low % kBlock);
    }
    const _Float16 *q[RM];
    const float *powers[RM], *rows[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int64_t r = m0 + 16 * i + col < a.M ? m0 + 16 * i + col : a.M - 1;
        if constexpr (LAID) {
            q[i] = f.w.q + r * f.w.ld;
            powers[i] = f.w.powers + r;
        } else {
            rows[i] = a.x + r * a.ldx;
        }
    }
    float4v acc[RM][RN];
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) acc[i][j] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    // Numbers 16 group .. of a block and 64 + 16 group .., eight an MFMA.
    for (int b = split; b < blocks; b += S) {
        const int64_t k = static_cast<int64_t>(b) * kBlock + 16 * group;
        half8 v[RN][4], x[RM][4];
        float power[RM], s[RN][2];
#pragma unroll
        for (int j = 0; j < RN; ++j) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int4v p = load_w(w[j], k + 64 * h, a.K);
                v[j][2 * h] = widen(p[0], p[1]);
                v[j][2 * h + 1] = widen(p[2], p[3]);
            }
            s[j][0] = scales[j][0][b];
            s[j][1] = GATED ? scales[j][1][b] : s[j][0];
        }
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            if constexpr (LAID) {
#pragma unroll
                for (int h = 0; h < 4; ++h) x[i][h] = *reinterpret_cast<const half8 *>(q[i] + k + 64 * (h / 2) + 8 * (h % 2));
                power[i] = powers[i][b * f.w.rows];
            } else {
                float4v u[8];
                uint32_t top = 0;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    u[c] = load_x(rows[i], k + 64 * (c / 4) + 4 * (c % 4), a.K);
#pragma unroll
                    for (int d = 0; d < 4; ++d) top = greater(top, magnitude(u[c][d]));
                }
                uint32_t other = top;
                swap16(top, other);
                top = greater(top, other);
                other = top;
                swap32(top, other);
                top = greater(top, other);
                const uint32_t e = power_of(top);
                const float scale = down(e);
                const bool finite = top < kInfinity;
#pragma unroll
                for (int h = 0; h < 4; ++h) x[i][h] = widen(four(u[2 * h], scale, finite), four(u[2 * h + 1], scale, finite));
                power[i] = finite ? up(e) : 1.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < RN; ++j) {
                float4v p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int h = 0; h < 4; ++h) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[j][h], x[i][h], p, 0, 0, 0);
                const float f0 = s[j][0] * power[i], f1 = s[j][1] * power[i];
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[i][j][c] = __builtin_fmaf(GATED && c >= across[j] ? f1 : f0, p[c], acc[i][j][c]);
            }
    }
    const int count = P * RM * 256;  // outputs of a workgroup, [tile][16 rows][row][column]
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j)
            *reinterpret_cast<float4v *>(sums + (split * RN + j) * count + (tile * RM + i) * 256 + col * 16 + 4 * group) = acc[i][j];
    lds_barrier();
    const auto place = [&](int at, int64_t &m, int &out) {
        m = m0 + 16 * ((at >> 8) % RM) + ((at >> 4) & 15);
        out = n0 + 16 * ((at >> 8) / RM) + (at & 15);
        return 1.0f;
    };
    write_outputs<GATED, 2>(a, sums, S, RN * count, count, tid, columns, place, kThreads);
}

template <bool GATED, bool LAID, int RM>
hipError_t launch_rows(RowsArgs f, hipStream_t stream) {
    constexpr int kLds = kWaves * RM * (GATED ? 2 : 1) * 1024;
    const int64_t columns = GATED ? f.a.half : f.a.N;
    const int64_t waves = static_cast<int64_t>(compute_units()) * kWaves, blocks = ceil_div(f.a.K, kF8Block);
    const int64_t rows = ceil_div(f.a.M, 16 * RM);
    int splits = 1;
    while (splits < kWaves && 2 * splits <= blocks && ceil_div(columns, 16) * rows * splits < waves) splits *= 2;
    f.splits = splits;
    f.column_blocks = static_cast<uint32_t>(ceil_div(columns, 16 * (kWaves / splits)));
    SDHIP_LAUNCH((f8_rows_kernel<GATED, LAID, RM>), dim3(static_cast<uint32_t>(f.column_blocks * rows)), dim3(kThreads), kLds, stream, f);
    return hipGetLastError();
}

// ------------------------------------------------------------------ the choice

// Which kernels a product takes, numbered as the f8_form tuning asks for them.
enum class Form { few = 1, rows };

Form form_of(int64_t M) { return M <= 16 ? Form::few : Form::rows; }

hipError_t lay_out(const F8Args &a, const F8Work &w, hipStream_t stream) {
    const int64_t blocks = w.ld / kF8Block, groups = blocks * a.M, x_grid = ceil_div(groups, kOperandThreads / 16);
    const int64_t w_grid = w.w != nullptr ? ceil_div(a.N * (w.ld / 16), kOperandThreads) : 0;
    const OperandsArgs o{a, w, static_cast<uint32_t>(blocks), static_cast<uint32_t>(groups), static_cast<uint32_t>(x_grid)};
    SDHIP_LAUNCH(f8_operands_kernel, dim3(static_cast<uint32_t>(x_grid + w_grid)), dim3(kOperandThreads), 0, stream, o);
    return hipGetLastError();
}

template <bool GATED>
hipError_t launch_form(const F8Args &a, bool whole, void *work, hipStream_t stream) {
    const Form form = form_of(a.M);
    if (form == Form::few) return launch_rows<GATED, false, 1>(RowsArgs{a, F8Work{}, 1, 0}, stream);
    const F8Work w = work_of(a.M, a.N, a.K, false, work);
    if (const hipError_t e = lay_out(a, w, stream); e != hipSuccess) return e;
    return launch_rows<GATED, true, 2>(RowsArgs{a, w, 1, 0}, stream);
}

}  // namespace

size_t f8_work_size(int64_t M, int64_t N, int64_t K, bool whole) {
    const Form form = form_of(M);
    return form == Form::few ? 0 : work_of(M, N, K, false, nullptr).bytes;
}

hipError_t launch_f8_mul_mat(const F8Args &a, bool whole, void *work, hipStream_t stream) {
    KernelScope scope(a.half ? "f8.gated" : "f8", stream);
    return a.half ? launch_form<true>(a, whole, work, stream) : launch_form<false>(a, whole, work, stream);
}

}  // namespace sdhip
