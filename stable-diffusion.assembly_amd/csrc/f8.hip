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

#include <type_traits>

#include "f8.h"
#include "host.h"
#include "outputs.h"
#include "profile.h"

namespace sdhip {

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));

constexpr int kBlock = static_cast<int>(kF8Block);
constexpr int kLeast = -101 + 127;  // e's least, biased as an exponent's bits
constexpr uint32_t kInfinity = 0x7f800000u;

// ------------------------------------------------------------------ numbers

// e's bits, biased by 127, for a greatest magnitude of these bits: 448 is 1.75 x
// 2^8.
__device__ __forceinline__ uint32_t power_of(uint32_t greatest) {
    const int e = static_cast<int>((greatest + 0x1fffffu) >> 23) - 8;
    return static_cast<uint32_t>(e > kLeast ? e : kLeast);
}

// 2^e and 2^-e.
__device__ __forceinline__ float up(uint32_t e) { return __builtin_bit_cast(float, e << 23); }
__device__ __forceinline__ float down(uint32_t e) { return __builtin_bit_cast(float, (254 - e) << 23); }

// The greatest magnitude of a group's eight numbers of each of 16 lanes, as bits, on
// all of them: of NaN among them nothing is seen.
__device__ __forceinline__ uint32_t greatest(const float4v &u, const float4v &v) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __builtin_fmaxf(m, __builtin_fabsf(u[i]));
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __builtin_fmaxf(m, __builtin_fabsf(v[i]));
    uint32_t top = __builtin_bit_cast(uint32_t, m);
    const auto greater = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    top = greater(top, __builtin_amdgcn_update_dpp(0, top, 0xb1, 0xf, 0xf, true));   // lanes i ^ 1
    top = greater(top, __builtin_amdgcn_update_dpp(0, top, 0x4e, 0xf, 0xf, true));   // i ^ 2
    top = greater(top, __builtin_amdgcn_update_dpp(0, top, 0x141, 0xf, 0xf, true));  // 8 lanes mirrored
    return greater(top, __builtin_amdgcn_update_dpp(0, top, 0x140, 0xf, 0xf, true));  // 16 lanes mirrored
}

// Eight numbers of E4M3 as FP16.
__device__ __forceinline__ half8 widen(int low, int high) {
    const half2v a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(low, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(low, 1.0f, true);
    const half2v c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(high, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(high, 1.0f, true);
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Four numbers times `scale` as E4M3.
__device__ __forceinline__ int four(const float4v &v, float scale) {
    const int r = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * scale, v[1] * scale, 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * scale, v[3] * scale, r, true);
}

// A lane's eight numbers of a group as q, and the group's 2^e.  An infinity makes them
// all NaN; a NaN stays one.
__device__ __forceinline__ int2 held(const float4v &u, const float4v &v, float &power) {
    const uint32_t top = greatest(u, v), e = power_of(top);
    const float scale = top < kInfinity ? down(e) : __builtin_nanf("");
    power = up(e);
    return make_int2(four(u, scale), four(v, scale));
}

// Four of a row's K numbers from k on, of the last four there are where those end
// before; rows of fewer than four number by number, 0 past their end.
__device__ __forceinline__ float4v load_x(const float *row, int k, int K) {
    if (K >= 4) return load4(row + (k + 4 <= K ? k : K - 4));
    float4v v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (k + i < K) v[i] = row[k + i];
    return v;
}

// What load_x gave at k as the numbers from there on, 0 past the row's end.
__device__ __forceinline__ float4v ended_x(const float4v &v, int k, int K) {
    const int past = k + 4 - K;  // numbers that lie before k, and are wanted of none past K
    if (!__any(past > 0) || K < 4 || past <= 0) return v;
    return past == 1 ? float4v{v[1], v[2], v[3], 0.0f} : past == 2 ? float4v{v[2], v[3], 0.0f, 0.0f}
                                                    : past == 3 ? float4v{v[3], 0.0f, 0.0f, 0.0f} : float4v{0.0f, 0.0f, 0.0f, 0.0f};
}

// 16 of a row's K weights from k on, of the last 16 there are where those end
// before: of what follows a row nothing is read, since it may be no memory.  Rows of
// fewer than 16 are read byte by byte, 0 past their end.
__device__ __forceinline__ int4v load_w(const uint8_t *row, int k, int K) {
    int4v v = {0, 0, 0, 0};
    if (K >= 16) {
        __builtin_memcpy(&v, row + (k + 16 <= K ? k : K - 16), 16);
    } else {
        uint64_t low = 0, high = 0;
#pragma unroll 1
        for (int i = k; i < K; ++i) {
            const uint64_t byte = static_cast<uint64_t>(row[i]) << (8 * (i & 7));
            low |= i < 8 ? byte : 0;
            high |= i < 8 ? 0 : byte;
        }
        const uint64_t q[2] = {low, high};
        __builtin_memcpy(&v, q, 16);
    }
    return v;
}

// What load_w gave at k as the weights from there on, 0 past the row's end.
__device__ __forceinline__ int4v ended_w(int4v v, int k, int K) {
    const int past = k + 16 - K;  // bytes that lie before k, and are wanted of none past K
    if (K < 16 || past <= 0) return v;
    if (past >= 16) return int4v{0, 0, 0, 0};
    uint64_t q[2];
    __builtin_memcpy(q, &v, 16);
    const int bits = 8 * (past & 7);
    if (past >= 8) {
        q[0] = q[1];
        q[1] = 0;
    }
    if (bits) {
        q[0] = q[0] >> bits | q[1] << (64 - bits);
        q[1] >>= bits;
    }
    __builtin_memcpy(&v, q, 16);
    return v;
}

// ------------------------------------------------------------------ the work buffer

// x's q by halves of a block, zeros past K: [half][row][64]; its 2^e, [block][row]; the
// weights as rows of whole blocks, zeros past K, where theirs are at other places than
// multiples of 16 bytes.
struct F8Work {
    uint8_t *q;
    float *powers;
    uint8_t *w;
    int64_t ld;    // K rounded up to whole blocks
    int64_t rows;  // M rounded up to whole tiles
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
    w.q = reinterpret_cast<uint8_t *>(take(w.rows * w.ld));
    w.powers = reinterpret_cast<float *>(take(4 * w.rows * (w.ld / kF8Block)));
    if (weights) w.w = reinterpret_cast<uint8_t *>(take(N * w.ld));
    w.bytes = at;
    return w;
}

constexpr int kOperandThreads = 256;

struct OperandsArgs {
    F8Args a;
    F8Work w;
    uint32_t across, tiles;  // tiles of x: along K, and all
    uint32_t x_grid;         // the workgroups that lay out x
};

// Tiles of 4 rows of x by 4 blocks of K, a group by 16 lanes, 8 numbers each: pieces of
// 2 KB read and 256 bytes written (16 rows by a block: 4096 x 4096 28 us, so
// 19; 1976 x 5120 10.5 both ways).
// Behind them the weights' rows, 16 numbers a lane.
__global__ __launch_bounds__(kOperandThreads) void f8_operands_kernel(OperandsArgs o) {
    const F8Args &a = o.a;
    if (blockIdx.x >= o.x_grid) {
        const int64_t pieces = o.w.ld / 16, all = pieces * a.N, step = static_cast<int64_t>(gridDim.x - o.x_grid) * kOperandThreads;
        for (int64_t i = static_cast<int64_t>(blockIdx.x - o.x_grid) * kOperandThreads + threadIdx.x; i < all; i += step) {
            const int64_t n = i / pieces;
            const int k = static_cast<int>(i - n * pieces) * 16, K = static_cast<int>(a.K);
            *reinterpret_cast<int4v *>(o.w.w + n * o.w.ld + k) = ended_w(load_w(a.w + n * a.row_bytes, k, K), k, K);
        }
        return;
    }
    const uint32_t team = threadIdx.x / 16, part = threadIdx.x & 15, blocks = static_cast<uint32_t>(o.w.ld / kBlock);
    for (uint32_t g = blockIdx.x; g < o.tiles; g += o.x_grid) {
        const uint32_t down = g / o.across;
        const int64_t m = 4 * static_cast<int64_t>(down) + team / 4, b = 4 * (g - down * o.across) + team % 4;
        if (m >= a.M || b >= blocks) continue;  // the 16 lanes of a group together
        const int k = static_cast<int>(b) * kBlock + 8 * static_cast<int>(part), K = static_cast<int>(a.K);
        const float *row = a.x + m * a.ldx;
        const float4v u = ended_x(load_x(row, k, K), k, K), v = ended_x(load_x(row, k + 4, K), k + 4, K);
        float power;
        const int2 q = held(u, v, power);
        *reinterpret_cast<int2 *>(o.w.q + ((2 * b + part / 8) * o.w.rows + m) * 64 + 8 * (part & 7)) = q;
        if (part == 0) o.w.powers[b * o.w.rows + m] = power;
    }
}

// ------------------------------------------------------------------ few rows

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;

struct FewArgs {
    F8Args a;
    int32_t splits;  // of K, a wave each; the other waves take further columns
    int32_t chunk;   // blocks of K whose x is in LDS at a time
    int32_t row;     // bytes of a row of it
    uint32_t column_blocks;
};

// A wave's blocks of the weights under way: as many as 128 registers hold, for two
// workgroups a CU.
constexpr int few_ahead(int rm) { return rm > 1 ? 2 : 3; }

// A workgroup takes 16 RM rows of x and kWaves / splits tiles of 16 rows of the
// weights (with GATED half of them of each half), a wave a tile and every splits-th
// block of K.  x is brought to E4M3 in it, a group by 16 lanes, LOADS of them under
// way, and kept in LDS in FP16 with the groups' powers, by chunks of K where it is
// long; the weights come straight from memory into registers, few_ahead blocks of a
// wave's under way, 64 bytes of a row side by side in a load.  The splits' sums are
// joined in LDS.  TAIL: K ends within a block, which is taken apart from the whole ones.
// Of 1 x 4096 -> 16384 the weights' bytes are the bound (14.5 us, 4.6 TB/s); at 1280 ->
// 1280 (4.4 us) the launch and what waits for one another: x, its greatest, a barrier,
// the products and the splits' sums.
template <bool GATED, bool TAIL, int RM, int LOADS>
__global__ __launch_bounds__(kThreads, LOADS > 2 ? 2 : 4) void f8_few_kernel(FewArgs f) {
    const F8Args &a = f.a;
    constexpr int kRows = 16 * RM, kAhead = few_ahead(RM);
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, group = lane >> 4;
    const int S = f.splits, P = kWaves / S;
    const int outs = GATED ? P / 2 : P;  // tiles of the output
    const int split = wave & (S - 1), second = GATED && wave / S >= outs, tile = wave / S - (second ? outs : 0);
    const uint32_t row_block = blockIdx.x / f.column_blocks;
    const int64_t m0 = static_cast<int64_t>(row_block) * kRows;
    const int rows = static_cast<int>(a.M - m0 < kRows ? a.M - m0 : kRows);
    const int columns = static_cast<int>(GATED ? a.half : a.N);
    const int n0 = static_cast<int>(blockIdx.x - row_block * f.column_blocks) * (16 * outs);
    const int K = static_cast<int>(a.K), blocks = (K + kBlock - 1) / kBlock;
    const int n = n0 + 16 * tile;

    // Groups of x, 32 at a time by the workgroup, LOADS such passes' loads together; the
    // row of group g by a product that is exact for the few thousands there are.
    const auto row_of = [](int g, float inverse) { return static_cast<int>((static_cast<float>(g) + 0.5f) * inverse); };
    const int team = tid >> 4, part = tid & 15;
    float *powers = reinterpret_cast<float *>(lds + rows * f.row);  // [row][block of the chunk]
    const auto x_row_of = [&](int r) {
        return a.x + m0 * K + static_cast<uint64_t>(static_cast<uint32_t>(r)) * static_cast<uint32_t>(K);
    };
    struct Numbers {
        float4v v[LOADS][2];
    };
    const auto load_groups = [&](int b0, int count, int first, Numbers &x) {
        const float inverse = 1.0f / static_cast<float>(count);
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int g = first + 32 * u + team, r = row_of(g, inverse), k = (b0 + g - r * count) * kBlock + 8 * part;
            const float *from = x_row_of(r < rows ? r : rows - 1) + k;
            x.v[u][0] = load4(from);
            x.v[u][1] = load4(from + 4);
        }
    };
    const auto store_group = [&](int r, int b, int2 q, float power) {
        *reinterpret_cast<half8 *>(lds + r * f.row + b * (2 * kBlock) + 16 * part) = widen(q.x, q.y);
        if (part == 0) powers[r * f.chunk + b] = power;
    };
    const auto store_groups = [&](int count, int first, const Numbers &x) {
        const float inverse = 1.0f / static_cast<float>(count);
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const int g = first + 32 * u + team, r = row_of(g, inverse);
            float power;
            const int2 q = held(x.v[u][0], x.v[u][1], power);
            if (r < rows) store_group(r, g - r * count, q, power);
        }
    };
    // The whole blocks of a chunk from b0 on.
    const auto whole_of = [&](int b0) {
        const int whole = K / kBlock - b0;
        return whole < f.chunk ? whole : f.chunk;
    };
    Numbers begun;
    if (!TAIL || whole_of(0) > 0) load_groups(0, whole_of(0), 0, begun);

    // The lane's row of the weights; the scales of its first output and of its last,
    // which with GATED lie in two blocks at most, `across` of them in the first.
    const int64_t from = second ? columns : 0;
    const uint8_t *w = a.w + (from + (n + col < columns ? n + col : columns - 1)) * a.row_bytes;
    const int64_t low = from + (n + 4 * group < columns ? n + 4 * group : columns - 1), high = low + 3 < a.N ? low + 3 : a.N - 1;
    const float *scales[2] = {a.scales + low / kBlock * a.ld_scales, a.scales + high / kBlock * a.ld_scales};
    const int across = kBlock - static_cast<int>(low % kBlock);
    struct Weights {
        int4v q[2];  // numbers 16 group .. of a block and 64 + 16 group ..
        float s[2];
    };
    const auto load_weights = [&](int b, Weights &o) {
        if (b >= blocks) return;
        const int k = b * kBlock + 16 * group;
        if (TAIL && (b + 1) * kBlock > K) {
            o.q[0] = load_w(w, k, K);
            o.q[1] = load_w(w, k + 64, K);
        } else {
            __builtin_memcpy(&o.q[0], w + k, 16);
            __builtin_memcpy(&o.q[1], w + k + 64, 16);
        }
        o.s[0] = scales[0][b];
        o.s[1] = GATED ? scales[1][b] : o.s[0];
    };
    Weights weights[kAhead];
#pragma unroll
    for (int d = 0; d < kAhead; ++d) load_weights(split + d * S, weights[d]);

    // A lane's rows of x, or the last there is.
    const char *x_row[RM];
    const float *x_power[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int r = 16 * i + col < rows ? 16 * i + col : rows - 1;
        x_row[i] = lds + r * f.row + 32 * group;
        x_power[i] = powers + r * f.chunk;
    }
    float4v acc[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i) acc[i] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    if (!TAIL || whole_of(0) > 0) store_groups(whole_of(0), 0, begun);
    for (int b0 = 0;;) {
        const int count = blocks - b0 < f.chunk ? blocks - b0 : f.chunk, whole = whole_of(b0);
#pragma unroll 1
        for (int first = b0 == 0 ? 32 * LOADS : 0; first < rows * whole; first += 32 * LOADS) {
            Numbers x;
            load_groups(b0, whole, first, x);
            store_groups(whole, first, x);
        }
        if (TAIL && whole < count && team < rows) {
            const int k = (blocks - 1) * kBlock + 8 * part;
            const float *from = x_row_of(team);
            float power;
            const int2 q = held(ended_x(load_x(from, k, K), k, K), ended_x(load_x(from, k + 4, K), k + 4, K), power);
            store_group(team, whole, q, power);
        }
        lds_barrier();
#pragma unroll 1
        for (int b1 = split; b1 < count; b1 += kAhead * S) {
#pragma unroll
            for (int d = 0; d < kAhead; ++d) {
                const int b = b1 + d * S;
                if (b >= count) continue;
                if (TAIL && (b0 + b + 1) * kBlock > K) {  // a shorter block, the last
                    const int k = (b0 + b) * kBlock + 16 * group;
                    weights[d].q[0] = ended_w(weights[d].q[0], k, K);
                    weights[d].q[1] = ended_w(weights[d].q[1], k + 64, K);
                }
                half8 v[4];
#pragma unroll
                for (int h = 0; h < 4; ++h) v[h] = widen(weights[d].q[h / 2][2 * (h % 2)], weights[d].q[h / 2][2 * (h % 2) + 1]);
                const float s[2] = {weights[d].s[0], weights[d].s[1]};
                load_weights(b0 + b + kAhead * S, weights[d]);
#pragma unroll
                for (int i = 0; i < RM; ++i) {
                    half8 x[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h)
                        x[h] = *reinterpret_cast<const half8 *>(x_row[i] + b * (2 * kBlock) + 128 * (h / 2) + 16 * (h % 2));
                    float4v p = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int h = 0; h < 4; ++h) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[h], x[h], p, 0, 0, 0);
                    const float power = x_power[i][b], f0 = s[0] * power, f1 = s[1] * power;
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[i][c] = __builtin_fmaf(GATED && c >= across ? f1 : f0, p[c], acc[i][c]);
                }
            }
        }
        lds_barrier();  // the chunk is read
        b0 += f.chunk;
        if (b0 >= blocks) break;
    }
    float *sums = reinterpret_cast<float *>(lds);
    const int count = outs * RM * 256;  // outputs of a workgroup, [tile][16 rows][row][column]
#pragma unroll
    for (int i = 0; i < RM; ++i)
        *reinterpret_cast<float4v *>(sums + (GATED ? 2 * split + second : split) * count + (tile * RM + i) * 256 + col * 16 + 4 * group) = acc[i];
    lds_barrier();
    const auto place = [&](int at, int64_t &m, int &out) {
        m = m0 + 16 * ((at >> 8) % RM) + ((at >> 4) & 15);
        out = n0 + 16 * ((at >> 8) / RM) + (at & 15);
        return 1.0f;
    };
    write_outputs<GATED, 2>(a, sums, S, (GATED ? 2 : 1) * count, count, tid, columns, place, kThreads);
}

// Splits of K until every wave of the device has one; `halves`, 2 of the gated.
int few_splits(int64_t M, int64_t columns, int64_t K, int64_t rows, int halves) {
    const int64_t waves = static_cast<int64_t>(compute_units()) * kWaves, blocks = ceil_div(K, kF8Block);
    const int64_t tiles = halves * ceil_div(columns, 16) * ceil_div(M, rows);
    int splits = 1;
    while (splits < kWaves / halves && 2 * splits <= blocks && tiles * splits < waves) splits *= 2;
    return splits;
}

template <bool GATED, bool TAIL, int RM, int LOADS>
hipError_t launch_few(FewArgs f, int64_t rows, int64_t row_blocks, hipStream_t stream) {
    constexpr int kSums = kWaves * RM * 1024, kMost = 160 * 1024;
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&f8_few_kernel<GATED, TAIL, RM, LOADS>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (attr != hipSuccess) return attr;
    const int64_t x = rows * (f.row + 4 * static_cast<int64_t>(f.chunk));
    SDHIP_LAUNCH((f8_few_kernel<GATED, TAIL, RM, LOADS>), dim3(static_cast<uint32_t>(f.column_blocks * row_blocks)), dim3(kThreads),
                 static_cast<uint32_t>(x > kSums ? x : kSums), stream, f);
    return hipGetLastError();
}

template <bool GATED, bool TAIL, int RM>
hipError_t few_rows(const F8Args &a, hipStream_t stream) {
    const int64_t columns = GATED ? a.half : a.N, blocks = ceil_div(a.K, kF8Block);
    const int64_t rows = a.M < 16 * RM ? a.M : 16 * RM, row_blocks = ceil_div(a.M, 16 * RM);
    const int splits = few_splits(a.M, columns, a.K, 16 * RM, GATED ? 2 : 1), outs = kWaves / splits / (GATED ? 2 : 1);
    // Whole rounds of the waves' blocks: all of K where that is 64 KB at most, else as
    // many as 64 KB hold, or one (100 KB of 16 rows, 133 of 32).
    const int64_t round = few_ahead(RM) * splits, bytes = 2 * kBlock + 4;
    const int64_t fit = (64 * 1024 / rows - 16) / bytes / round * round;
    const int64_t chunk = blocks < fit ? blocks : fit > round ? fit : round < blocks ? round : blocks;
    // Rows 16 bytes further apart than they are long, so that 16 read at once lie on
    // different banks.
    const FewArgs f{a, splits, static_cast<int32_t>(chunk), static_cast<int32_t>(chunk * (2 * kBlock) + 16),
                    static_cast<uint32_t>(ceil_div(columns, 16 * outs))};
    // All of a chunk's groups loaded together where a workgroup is alone on its CU;
    // else two passes, in the registers that leave room for another workgroup.
    const int64_t passes = ceil_div(rows * chunk, kThreads / 16);
    const bool alone = f.column_blocks * row_blocks <= compute_units();
    if (passes <= 1) return launch_few<GATED, TAIL, RM, 1>(f, rows, row_blocks, stream);
    if (passes <= 2 || !alone) return launch_few<GATED, TAIL, RM, 2>(f, rows, row_blocks, stream);
    return launch_few<GATED, TAIL, RM, 4>(f, rows, row_blocks, stream);
}

template <bool GATED, int RM>
hipError_t few_rows(const F8Args &a, hipStream_t stream) {
    return a.K % kF8Block != 0 ? few_rows<GATED, true, RM>(a, stream) : few_rows<GATED, false, RM>(a, stream);
}

// ------------------------------------------------------------------ many rows

// Both operands by tiles through LDS: a workgroup takes 64 WM rows of x by 64 WN
// of the weights (with GATED 32 WN of each half), waves 64 x 64 of them each, and WK
// blocks of K at a time, WK waves' sums joined at the end.  A stage is half a block
// of each, 64 numbers of a row, and the block's powers and scales.  Both are in LDS as
// E4M3, widened by each wave that reads them: of x in FP16 there the copies and the
// reads would be half as much again, and they weigh more than the vector operations
// saved (4096 x 4096 -> 16384: 588 us against 554).  A lane's 16 bytes are at a place
// of their row that spreads 16 rows read at once over LDS's banks.  kRing stages are in LDS, one
// read and the others under way (four: 1976 x 1280 -> 10240 71.6 us against 69.0).
//
// 4096 x 4096 -> 16384 takes 520 to 550 us, 1.0 PFLOP/s, where a library's product of
// FP16 takes 380 to 460, as the card and the numbers are: its MFMAs are busy 82% of the
// cycles at the 1.55 GHz that the card then runs, these 55% at 1.76, with 7.4 other vector operations a MFMA (4 that widen, 2 that
// add a block's sums) on the same ports, LDS read or written 75% of the MFMAs' time.
// Whole rounds of tiles are the rest: 1976 x 5120 -> 1280 has 160 for 256 CUs.
constexpr int kRing = 3;

template <int WM, int WN, int WK>
struct Tiles {
    static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves * WK;
    static constexpr int kX = 64 * WM, kW = 64 * WN;  // rows of the tiles
    static constexpr int kXBytes = 64 * kX, kWBytes = 64 * kW, kPowers = 4 * kX, kScales = 256;
    static constexpr int kPart = kXBytes + kWBytes + kPowers + kScales;  // of a block
    static constexpr int kStage = WK * kPart;
    static constexpr int kXCopies = 4 * WM / kWaves, kWCopies = 4 * WN / kWaves;  // a wave's, of 1 KB
    static constexpr int kSmallCopies = (WM + 1 + kWaves - 1) / kWaves;          // and of 256 bytes
    static constexpr int kCopies = kXCopies + kWCopies + kSmallCopies;
    static_assert(4 * WM % kWaves == 0 && 4 * WN % kWaves == 0);
    // WK waves' sums are joined in LDS.
    static constexpr int kSums = WK == 1 ? 0 : 16384 * kWaves * WK;
    static constexpr int kLds = kRing * kStage > kSums ? kRing * kStage : kSums;
};

struct TilesArgs {
    F8Args a;
    F8Work work;
    const uint8_t *w;  // rows at multiples of 16 bytes, of a multiple of 16 ...
    int64_t ldw;       // ... this far apart
    int32_t end;       // ... and this long
    uint32_t row_blocks, column_blocks;
};

// ENDS: the weights' rows end within a block.
template <bool GATED, bool ENDS, int WM, int WN, int WK>
__global__ __launch_bounds__(64 * WM * WN * WK, 2) void f8_tiles_kernel(TilesArgs t) {
    using L = Tiles<WM, WN, WK>;
    const F8Args &a = t.a;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wk = wave / L::kWaves, place = wave % L::kWaves, wm = place % WM, wn = place / WM;
    const int col = lane & 31, hf = lane >> 5;
    // Groups of 8 row blocks by all columns: those at work at once in an XCD share
    // their operands' panels in its L2 both ways.
    const uint32_t at = xcd_swizzle(blockIdx.x, t.row_blocks * t.column_blocks);
    const uint32_t group = at / (8 * t.column_blocks), in = at - group * (8 * t.column_blocks);
    const uint32_t high = t.row_blocks - 8 * group < 8 ? t.row_blocks - 8 * group : 8;
    const int64_t m0 = static_cast<int64_t>(8 * group + in % high) * L::kX;
    const int columns = static_cast<int>(GATED ? a.half : a.N);
    const int n0 = static_cast<int>(in / high) * (GATED ? L::kW / 2 : L::kW);
    const int blocks = static_cast<int>(t.work.ld / kBlock);
    const int stages = 2 * ((blocks + WK - 1) / WK);

    // Row r of the weights' tile: its column of the output, in which half.
    const auto column_of = [&](int r, int &second) {
        second = GATED ? (r >> 5) & 1 : 0;
        const int n = GATED ? n0 + 32 * (r >> 6) + (r & 31) : n0 + r;
        return n < columns ? n : columns - 1;
    };
    // 16 rows a copy, a row by 4 lanes, its 16 bytes in the order of their places in LDS.
    const int piece = 16 * ((lane & 3) ^ (lane >> 4));
    uint32_t x_offset[L::kXCopies], w_offset[L::kWCopies];
    const char *w_base[L::kWCopies];
    const char *x_base = reinterpret_cast<const char *>(t.work.q + m0 * 64);
    const int64_t x_step = t.work.rows * 64;
#pragma unroll
    for (int c = 0; c < L::kXCopies; ++c) {
        const int r = 16 * (place + L::kWaves * c) + (lane >> 2);
        x_offset[c] = 64 * r + piece;
    }
#pragma unroll
    for (int c = 0; c < L::kWCopies; ++c) {
        const int r = 16 * (place + L::kWaves * c) + (lane >> 2);
        int second;
        const int n = column_of(r, second);
        w_offset[c] = static_cast<uint32_t>((n - n0) * t.ldw + piece);
        const int half = GATED ? ((16 * (place + L::kWaves * c)) >> 5) & 1 : 0;
        w_base[c] = reinterpret_cast<const char *>(t.w + (static_cast<int64_t>(n0) + (half ? columns : 0)) * t.ldw);
    }
    // A lane's number of the small copies: of 64 of the rows' powers, or the scales of
    // each 32 rows of the weights' tile, the first's block's and the last's by lanes 2 i
    // and 2 i + 1; and how far apart those of the next block are.
    const float *small[L::kSmallCopies];
    int64_t small_step[L::kSmallCopies];
    uint32_t small_to[L::kSmallCopies];
#pragma unroll
    for (int c = 0; c < L::kSmallCopies; ++c) {
        const int r = place + L::kWaves * c;
        int second;
        const int i = (lane >> 1) % (L::kW / 32), n = column_of(32 * i, second);
        const int64_t first = n + (second ? columns : 0), last = first + 31 < a.N ? first + 31 : a.N - 1;
        small[c] = r < WM ? t.work.powers + m0 + 64 * r + lane : a.scales + (lane & 1 ? last : first) / kBlock * a.ld_scales;
        small_step[c] = r < WM ? t.work.rows : 1;
        small_to[c] = L::kXBytes + L::kWBytes + (r < WM ? 256 * r : L::kPowers);
    }
    char *part = lds + wk * L::kPart;
    const auto copy = [&](int s, int buffer) {
        // Past the last block it once more, and past the last stage.
        const int pair = (s < stages ? s : stages - 1) >> 1;
        const int b = pair * WK + wk < blocks ? pair * WK + wk : blocks - 1;
        const int64_t k = static_cast<int64_t>(b) * kBlock + 64 * (s & 1);
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds_address(part) + buffer * L::kStage);
#pragma unroll
        for (int c = 0; c < L::kXCopies; ++c) fetch16(x_base + (2 * b + (s & 1)) * x_step, x_offset[c], to + 1024 * (place + L::kWaves * c));
#pragma unroll
        for (int c = 0; c < L::kWCopies; ++c) {
            const uint32_t at = to + L::kXBytes + 1024 * (place + L::kWaves * c);
            // Past a row's end its beginning, by x's zeros: a NaN there is its column's
            // anyway.  (By a branch the copies are apart: 76 x 1344 -> 14027 17.7 us, so 15.8.)
            const bool last = ENDS && k + 64 > t.end;
            const int back = last && k + piece >= t.end ? static_cast<int>(k) + piece : 0;
            fetch16(w_base[c] + (last ? 0 : k), last ? w_offset[c] + static_cast<int>(k) - back : w_offset[c], at);
        }
#pragma unroll
        for (int c = 0; c < L::kSmallCopies; ++c) fetch4(small[c] + b * small_step[c], to + small_to[c]);
    };
#pragma unroll
    for (int s = 0; s < kRing; ++s) copy(s, s);

    float16v acc[4], p[4];  // tile k: rows of x 32 (k % 2) .., of the weights 32 (k / 2) ..
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = p[k] = float16v{};
    // Operand o is 32 rows of x (0, 1) or of the weights (2, 3): as they are in LDS, and
    // as FP16 for two MFMAs.
    struct Operands {
        int4v q[4];
        half8 v[4][2];
    };
    // Rows of the tiles as the MFMA's lanes read them: of a quarter of a block.
    const char *x_row = part + 64 * (64 * wm + col), *w_row = part + L::kXBytes + 64 * (64 * wn + col);
    const int turn = (col >> 2) & 3;
    const auto read = [&](Operands &o, int buffer, int u) {
        const int at = buffer * L::kStage + 16 * ((2 * u + hf) ^ turn);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            o.q[i] = *reinterpret_cast<const int4v *>(x_row + at + 64 * 32 * i);
            o.q[2 + i] = *reinterpret_cast<const int4v *>(w_row + at + 64 * 32 * i);
        }
    };
    const auto widen_one = [&](Operands &o, int i) {
        o.v[i][0] = widen(o.q[i][0], o.q[i][1]);
        o.v[i][1] = widen(o.q[i][2], o.q[i][3]);
        // Here, not where they are used.
        asm volatile("" : "+v"(o.v[i][0]), "+v"(o.v[i][1]));
    };
    // A block's powers and scales; GATED: the second half's rows may lie in two
    // blocks of the scales, `across` of them in the first.
    float power[2], scale_of[2][2];
    const int across = GATED ? kBlock - static_cast<int>((columns + n0 + 32 * wn) % kBlock) : kBlock;
    const auto read_scales = [&](int buffer) {
        const char *small = part + buffer * L::kStage + L::kXBytes + L::kWBytes;
        const float *scales = reinterpret_cast<const float *>(small + L::kPowers) + 4 * wn;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            power[i] = reinterpret_cast<const float *>(small)[64 * wm + 32 * i + col];
            scale_of[i][0] = scales[2 * i];
            scale_of[i][1] = scales[2 * i + 1];
        }
    };
    const auto add = [&](int k) {
        const float f = scale_of[k >> 1][0] * power[k & 1];
        if (GATED && k >= 2 && across < 32) {
            const float g = scale_of[k >> 1][1] * power[k & 1];
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[k][e] = __builtin_fmaf(tile_row(e) + 4 * hf < across ? f : g, p[k][e], acc[k][e]);
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[k][e] = __builtin_fmaf(f, p[k][e], acc[k][e]);
        }
    };
    // A quarter of a block: its products from registers while the next one's
    // operands are read and widened; with `ends` a tile's sums are added while the
    // next tile's are made, the last one's with the first of the next quarter
    // (`kept`).
    const auto quarter = [&](const Operands &now, Operands &next, int buffer, int u, auto begins, auto kept, auto ends) {
        read(next, buffer, u);
        __builtin_amdgcn_sched_barrier(0);
        const auto tile = [&](auto tile_) {
            constexpr int k = decltype(tile_)::value;
            p[k] = __builtin_amdgcn_mfma_f32_32x32x16_f16(now.v[2 + k / 2][0], now.v[k % 2][0], begins ? float16v{} : p[k], 0, 0, 0);
            p[k] = __builtin_amdgcn_mfma_f32_32x32x16_f16(now.v[2 + k / 2][1], now.v[k % 2][1], p[k], 0, 0, 0);
            if (k == 0 && kept) add(3);
            if (k > 0 && ends) add(k - 1);
            if (k == 1) widen_one(next, 0);
            if (k == 2) {
                widen_one(next, 2);
                widen_one(next, 1);
            }
            if (k == 3) widen_one(next, 3);
            // In this order: an MFMA and half of the other operations, twice.
            constexpr int others = (k == 0 ? decltype(kept)::value : decltype(ends)::value ? 1 : 0) * 17 + (k == 0 ? 0 : k == 2 ? 16 : 8);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, (others + 1) / 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, (others + 1) / 2, 0);
            __builtin_amdgcn_sched_barrier(0);
        };
        tile(std::integral_constant<int, 0>{});
        tile(std::integral_constant<int, 1>{});
        tile(std::integral_constant<int, 2>{});
        tile(std::integral_constant<int, 3>{});
    };
    int buffer = 0;
    fetched<(kRing - 1) * L::kCopies>();
    lds_barrier();
    Operands even, odd;
    read(even, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) widen_one(even, i);
    // Stage s is in registers or being read; the copies of the kRing - 2 after it are
    // under way, and once s is read those of the next take its buffer.
    const auto arrive = [&](int s) {
        fetched<(kRing - 2) * L::kCopies>();
        lds_barrier();  // every wave's copies of stage s + 1 are in, and stage s is read
        copy(s + kRing, buffer);
        buffer = buffer == kRing - 1 ? 0 : buffer + 1;
    };
    power[0] = power[1] = scale_of[0][0] = scale_of[0][1] = scale_of[1][0] = scale_of[1][1] = 0.0f;
    constexpr std::true_type yes{};
    constexpr std::false_type no{};
#pragma unroll 1
    for (int s = 0; s < stages; s += 2) {
        quarter(even, odd, buffer, 1, yes, yes, no);  // the block before's last tile, times 0 at first
        arrive(s);
        quarter(odd, even, buffer, 0, no, no, no);
        read_scales(buffer);
        if constexpr (WK > 1) {
            // Past the last block nothing is added (an infinite scale would make it NaN).
            const uint32_t keep = (s >> 1) * WK + wk < blocks ? 0xffffffffu : 0;
            const auto kept = [&](float v) { return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, v) & keep); };
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                power[i] = kept(power[i]);
                scale_of[i][0] = kept(scale_of[i][0]);
                scale_of[i][1] = kept(scale_of[i][1]);
            }
        }
        quarter(even, odd, buffer, 1, no, no, no);
        arrive(s + 1);
        quarter(odd, even, buffer, 0, no, no, yes);
    }
    add(3);
    fetched<0>();

    // The outputs, by rows of x a lane: of E of a tile's 16 registers, which are 4
    // columns each.
    constexpr int E = WK == 4 ? 8 : 16;
    const int64_t last = a.M - 1;
    const int base = n0 + (GATED ? 32 * wn : 64 * wn) + 4 * hf;
    const auto write = [&](int i, int e0, float (&v)[2][E]) {
        const int64_t m = m0 + 64 * wm + 32 * i + col, row = m < last ? m : last;
        // Column of number e of j's tile, and whether all of the tile's are there.
        const auto column = [&](int j, int e) { return base + (GATED ? 0 : 32 * j) + tile_row(e0 + e); };
        const auto full = [&](int j) { return n0 + (GATED ? 32 * wn : 64 * wn + 32 * j) + 32 <= columns; };
        const auto load = [&](const float *from, int64_t step, int j, float (&o)[E]) {
            if (step == 1 && full(j)) {
#pragma unroll
                for (int e = 0; e < E; e += 4) {
                    const float4v q = load4(from + column(j, e));
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[e + c] = q[c];
                }
            } else if (step == 0) {
                const float one = *from;
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = one;
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = from[(column(j, e) < columns ? column(j, e) : columns - 1) * step];
            }
        };
        if (!GATED && a.from_redirect) {
            float o[2][E];
#pragma unroll
            for (int j = 0; j < 2; ++j) load(a.y + row * a.ldy, 1, j, o[j]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) v[j][e] = o[j][e] + v[j][e];
        }
#pragma unroll 1
        for (int c = 0; c < a.chain.count; ++c) {
            const DevStep &st = a.chain.steps[c];
            if (st.kind == kSilu) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < E; ++e) v[j][e] = silu(v[j][e]);
                continue;
            }
            const float *from = st.operand;
            if (st.flat123) {
                from += row * st.nb[1];
            } else {
                uint32_t i1, i2, i3;
                split_index(static_cast<uint32_t>(row), static_cast<uint32_t>(a.ne1), static_cast<uint32_t>(a.ne2), i1, i2, i3);
                from += i1 * st.nb[1] + i2 * st.nb[2] + i3 * st.nb[3];
            }
            float o[2][E];
#pragma unroll
            for (int j = 0; j < 2; ++j) load(from + (GATED && j ? a.half * st.nb[0] : 0), st.nb[0], j, o[j]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) v[j][e] = st.kind == kAdd ? __fadd_rn(v[j][e], o[j][e]) : __fmul_rn(v[j][e], o[j][e]);
        }
        if (m > last) return;
        float *y = a.y + m * a.ldy;
#pragma unroll
        for (int j = 0; j < (GATED ? 1 : 2); ++j)
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                float4v q;
#pragma unroll
                for (int c = 0; c < 4; ++c) q[c] = GATED ? v[0][e + c] * gelu(v[1][e + c]) : v[j][e + c];
                if (full(j)) {
                    __builtin_memcpy(y + column(j, e), &q, 16);
                } else {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (column(j, e + c) < columns) y[column(j, e + c)] = q[c];
                }
            }
    };
    if constexpr (WK == 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float v[2][E];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) v[j][e] = acc[2 * j + i][e];
            write(i, 0, v);
        }
    } else {
        // [block][wave][tile][4 registers][lane]; a wave adds up a WK-th of them.
        lds_barrier();  // the last stage is read, and no copy is under way
        float4v *sums = reinterpret_cast<float4v *>(lds) + lane;
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                sums[64 * (((wk * L::kWaves + place) * 4 + k) * 4 + g)] = float4v{acc[k][4 * g], acc[k][4 * g + 1], acc[k][4 * g + 2], acc[k][4 * g + 3]};
        lds_barrier();
        const int i = WK == 2 ? wk : wk >> 1, g0 = WK == 2 ? 0 : 2 * (wk & 1);
        float v[2][E];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int g = 0; g < E / 4; ++g) {
                float4v q = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int b = 0; b < WK; ++b) q += sums[64 * (((b * L::kWaves + place) * 4 + 2 * j + i) * 4 + g0 + g)];
#pragma unroll
                for (int c = 0; c < 4; ++c) v[j][4 * g + c] = q[c];
            }
        write(i, 4 * g0, v);
    }
}

template <bool GATED, bool ENDS, int WM, int WN, int WK>
hipError_t launch_tiles(TilesArgs t, hipStream_t stream) {
    using L = Tiles<WM, WN, WK>;
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&f8_tiles_kernel<GATED, ENDS, WM, WN, WK>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, L::kLds);
    if (attr != hipSuccess) return attr;
    t.row_blocks = static_cast<uint32_t>(ceil_div(t.a.M, L::kX));
    t.column_blocks = static_cast<uint32_t>(GATED ? ceil_div(t.a.half, L::kW / 2) : ceil_div(t.a.N, L::kW));
    SDHIP_LAUNCH((f8_tiles_kernel<GATED, ENDS, WM, WN, WK>), dim3(t.row_blocks * t.column_blocks), dim3(L::kThreads), L::kLds, stream, t);
    return hipGetLastError();
}

// ------------------------------------------------------------------ the choice

// Which kernels a product takes, numbered as the f8_form tuning asks for them: the
// few rows' kernel by 16 rows or by 32, or tiles of 128 x 128 by four waves, of as many
// by eight's halves of K, of 64 x 128 by four's, of 64 x 64 by four's quarters.
enum class Form { few = 1, rows, tiles, tiles8, tiles64, tiles64x64 };

// Tiles' copies reach 128 rows of the weights by 32 bits of offset.
constexpr int64_t kTilesK = int64_t{1} << 22;

// Microseconds of the few rows' kernel by 16 RM rows: a launch and, for each round of
// workgroups over the CUs, a wave's blocks of the weights and all of its rows' x.
double few_time(int64_t M, int64_t columns, int64_t K, int rm, int halves) {
    const int splits = few_splits(M, columns, K, 16 * rm, halves);
    const int64_t blocks = ceil_div(K, kF8Block), groups = ceil_div(columns, 16 * (kWaves / splits / halves)) * ceil_div(M, 16 * rm);
    const double rounds = static_cast<double>(ceil_div(groups, compute_units()));
    const double rows = static_cast<double>(M < 16 * rm ? M : 16 * rm) / (16 * rm);
    const double own = static_cast<double>(ceil_div(blocks, splits)), x = rows * static_cast<double>(blocks);
    return rm == 1 ? 4.0 + rounds * (0.4 + 0.5 * own + 0.12 * x) : 4.4 + rounds * (0.8 + 0.6 * own + 0.27 * x);
}

// Tiles, the smallest of which there are no more than CUs, else the largest: of 1280
// columns and K 1280, us by 64 x 64 | 64 x 128 | 128 x 128: 768 rows 13.8 | 14.8 | 18.9,
// 1024 20.9 | 15.3 | 19.6, 8192 94 | 56 | 50.  Of the largest no more than CUs too, so
// one on each, and of a long K by eight waves: 2048 rows of 5120 to 1280 columns 51.7 by
// eight, 54.5 by four, 1024 of 320 to 2560 15.4 and 13.4.  Or a kernel of few rows, where that takes
// less by the times of a launch fitted to 28 such shapes, of 1 to 8192 rows (the rule
// is 1% slower than the best choice in the mean, 20% at most): of K 640 to 640 columns
// by 16 rows | 32 | tiles: 160 rows 5.3 | 6.4 | 10.3, 384 7.3 | 6.7 | 10.5, 1536 - | 13.0 |
// 11.9; of K 4096 to 4096 columns 32 rows 14.0 | 15.8 | -, 64 17.7 | 19.4 | 17.6.
Form form_of(int64_t M, int64_t N, int64_t K, bool gated) {
    const int halves = gated ? 2 : 1, asked = tuning().f8_form;
    const int64_t columns = N / halves;
    // The few rows' kernel takes a wave for 16 x 16 outputs, of the 2^26 a launch counts.
    const bool fits = (M / 16 + 1) * (N / 16 + 8) < (int64_t{1} << 25);
    if (asked > 0 && (asked <= 2 ? fits : K <= kTilesK)) return static_cast<Form>(asked);
    const double blocks = static_cast<double>(ceil_div(K, kF8Block));
    const auto tiles = [&](int64_t x, int64_t w) { return ceil_div(M, x) * ceil_div(columns, w / halves); };
    Form form = Form::tiles;
    double least = 8.2 + 0.5e-6 * static_cast<double>(M) * static_cast<double>(K);  // x is laid out
    if (tiles(64, 64) <= compute_units()) {
        form = Form::tiles64x64;
        least += 0.3 * blocks;
    } else if (tiles(64, 128) <= compute_units()) {
        form = Form::tiles64;
        least += 0.5 * blocks;
    } else {
        if (tiles(128, 128) <= compute_units() && K >= 2048) form = Form::tiles8;
        least += 0.9 * blocks * static_cast<double>(ceil_div(tiles(128, 128), 2 * compute_units()));
    }
    if (!fits) return form;
    const double few = few_time(M, columns, K, 1, halves), rows = few_time(M, columns, K, 2, halves);
    if (K <= kTilesK && least <= few && least <= rows) return form;
    return few <= rows ? Form::few : Form::rows;
}

bool by_tiles(Form form) { return form != Form::few && form != Form::rows; }

hipError_t lay_out(const F8Args &a, const F8Work &w, hipStream_t stream) {
    // 2^20 workgroups of each at most, of the 2^32 threads that a launch counts.
    const auto most = [](int64_t n) { return n < (1 << 20) ? n : 1 << 20; };
    const int64_t across = ceil_div(w.ld / kF8Block, 4), tiles = across * ceil_div(a.M, 4), x_grid = most(tiles);
    const int64_t w_grid = w.w != nullptr ? most(ceil_div(a.N * (w.ld / 16), kOperandThreads)) : 0;
    const OperandsArgs o{a, w, static_cast<uint32_t>(across), static_cast<uint32_t>(tiles), static_cast<uint32_t>(x_grid)};
    SDHIP_LAUNCH(f8_operands_kernel, dim3(static_cast<uint32_t>(x_grid + w_grid)), dim3(kOperandThreads), 0, stream, o);
    return hipGetLastError();
}

// Tiles whose weights' rows end within a block have kernels of their own: what their
// last copies take on costs the others 3 to 6% (4096 x 4096 -> 16384 582 us, so 600),
// and weights laid out first as much as the product (76 x 1344 -> 14027 25 us, so 15.8).
template <bool GATED, bool ENDS>
hipError_t launch_tiles(Form form, const TilesArgs &t, hipStream_t stream) {
    switch (form) {
    case Form::tiles8:
        return launch_tiles<GATED, ENDS, 2, 2, 2>(t, stream);
    case Form::tiles64:
        return launch_tiles<GATED, ENDS, 1, 2, 2>(t, stream);
    case Form::tiles64x64:
        return launch_tiles<GATED, ENDS, 1, 1, 4>(t, stream);
    default:
        return launch_tiles<GATED, ENDS, 2, 2, 1>(t, stream);
    }
}

template <bool GATED>
hipError_t launch_form(const F8Args &a, bool whole, void *work, hipStream_t stream) {
    const Form form = form_of(a.M, a.N, a.K, GATED);
    if (form == Form::few) return few_rows<GATED, 1>(a, stream);
    if (form == Form::rows) return few_rows<GATED, 2>(a, stream);
    const F8Work w = work_of(a.M, a.N, a.K, !whole, work);
    if (const hipError_t e = lay_out(a, w, stream); e != hipSuccess) return e;
    const TilesArgs t{a, w, whole ? a.w : w.w, whole ? a.row_bytes : w.ld, static_cast<int32_t>(whole ? a.K : w.ld), 0, 0};
    return t.end % kBlock != 0 ? launch_tiles<GATED, true>(form, t, stream) : launch_tiles<GATED, false>(form, t, stream);
}

}  // namespace

size_t f8_work_size(int64_t M, int64_t N, int64_t K, bool whole) {
    // Enough for the product and for the gated one.
    const bool tiles = by_tiles(form_of(M, N, K, false)) || (N % 2 == 0 && by_tiles(form_of(M, N, K, true)));
    return tiles ? work_of(M, N, K, !whole, nullptr).bytes : 0;
}

hipError_t launch_f8_mul_mat(const F8Args &a, bool whole, void *work, hipStream_t stream) {
    KernelScope scope(a.half ? "f8.gated" : "f8", stream);
    return a.half ? launch_form<true>(a, whole, work, stream) : launch_form<false>(a, whole, work, stream);
}

}  // namespace sdhip
