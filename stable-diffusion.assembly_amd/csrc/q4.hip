// MUL_MAT of weights in ggml's 4-bit blocks (Q4_0, Q4_1): each block of 32
// weights along K is a half-precision scale d, with Q4_1 a half-precision
// least value m, and 16 bytes, byte j holding number j in its low four bits
// and number 16 + j in its high ones.  Both types are one:
//     w = d (q - 8) + c,   c = 0 (Q4_0) or m + 8 d (Q4_1),
// so that a block's part of an output is d sum((q - 8) x) + c sum(x), q - 8 a
// whole number of -8 .. 7.
//
// The products are of FP16 on the MFMA: q - 8 is exact in it, and x is taken
// in two parts, hi = fp16(x 2^e) and lo = fp16(x 2^e - hi), with e bringing
// its row's greatest number to [2^14, 2^15): off by 2^-22 of a number at most, or
// below 2^-17 of the greatest, where half a step of lo is 2^-25, by 2^-39 of that.
// A block's 32 products fill one v_mfma_f32_16x16x32_f16 (two with both parts),
// whose sums in single precision are then scaled by d and added up; so no weight
// is rounded.  Q4_1's roundings are those of its two sums, |d (q - 8)| + |c| < 2.1
// max(|m|, |m + 15 d|) a number of x, of its own weight or not: with a channel
// 2^12 as great as the others and a weight of 0 there (q = 0, m = 0) the output is
// off by up to 1.4e-5 of the others' products, where q = 8 leaves 4e-8.  An offset
// next to a number of each block's own (c = m + z d, z from m / d) would hold each
// weight's products to 3 times itself, but costs few rows 6 to 20 % (one of 4096
// -> 16384 11.6 us, so 14.2).

#include <cmath>

#include "host.h"
#include "outputs.h"
#include "profile.h"
#include "q4.h"

namespace sdhip {

namespace {

// ------------------------------------------------------------------ blocks

// The 8 numbers q - 8 of a word's nibbles as FP16, by 1024 + q and 1024 + 16 q
// (a nibble in the last bits, or those four above, of 1024's mantissa), all
// exact: numbers 0, 2 (low nibbles), 16, 18 (high), 1, 3, 17, 19 of the four
// bytes' eight, the order that the columns of x are held in too.
// `magic` is kMagic in a vector register: a mask and it in one instruction.
constexpr uint32_t kMagic = 0x64006400u;
__device__ __forceinline__ half8 widen(uint32_t word, uint32_t magic) {
    typedef _Float16 half2 __attribute__((ext_vector_type(2)));
    const half2 low = {-1032, -1032}, high = {-72, -72}, down = {0.0625f, 0.0625f};
    const uint32_t odd = word >> 8;
    const half2 a = __builtin_bit_cast(half2, (word & 0x000f000fu) | magic) + low;
    const half2 b = __builtin_bit_cast(half2, (word & 0x00f000f0u) | magic) * down + high;
    const half2 c = __builtin_bit_cast(half2, (odd & 0x000f000fu) | magic) + low;
    const half2 e = __builtin_bit_cast(half2, (odd & 0x00f000f0u) | magic) * down + high;
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
}

// ------------------------------------------------------------------ x

// The power of two that brings a row's greatest magnitude (its bits) to
// [2^14, 2^15), as the bits of its exponent; 2^126 at most, so that the power
// that takes it back is a normal number.
__device__ __forceinline__ uint32_t scale_exponent(uint32_t greatest) {
    const uint32_t e = greatest >> 23;
    return 268 - e < 253 ? 268 - e : 253;
}

__device__ __forceinline__ float power(uint32_t exponent) { return __builtin_bit_cast(float, exponent << 23); }

// The greater magnitude of the wave's lanes, on all of them: within rows of
// 16 lanes by DPP, across them by swaps.
__device__ __forceinline__ uint32_t wave_greatest(uint32_t v) {
    const auto up = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    v = up(v, __builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, true));   // lanes i ^ 1
    v = up(v, __builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, true));   // i ^ 2
    v = up(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true));  // 8 lanes mirrored
    v = up(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true));  // 16 lanes mirrored
    uint32_t a = v, b = v;
    swap16(a, b);
    v = up(a, b);
    a = v;
    b = v;
    swap32(a, b);
    return up(a, b);
}

// Two parts of 8 numbers of x, low[0 .. 3] and high[0 .. 3] being 4 g .. and
// 16 + 4 g .. of a block, in widen's order.  An infinity is all in hi: its lo
// would be a NaN.
__device__ __forceinline__ void split8(const float4v &low, const float4v &high, float scale, half8 &hi, half8 &lo) {
    const float v[8] = {low[0], low[2], high[0], high[2], low[1], low[3], high[1], high[3]};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float s = v[i] * scale;
        hi[i] = static_cast<_Float16>(s);
        const float rest = s - static_cast<float>(hi[i]);
        lo[i] = static_cast<_Float16>(__builtin_isinf(s) ? 0.0f : rest);
    }
}

// The greatest magnitude of four numbers, as bits.
__device__ __forceinline__ uint32_t magnitude(const float4v &v) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t p = __builtin_bit_cast(uint32_t, static_cast<float>(v[k])) & 0x7fffffffu;
        m = m > p ? m : p;
    }
    return m;
}

constexpr int kFewThreads = 512;

// ------------------------------------------------------------------ few rows

// Up to 16 rows of x a workgroup.  It takes P tiles of 16 rows of the weights
// (with GATED, P / 2 of each half) by S splits of K, a wave each, 8 at most; a
// split is every S-th unit of 8 blocks, and the splits' sums are added at the
// end in their order.
//
// What bounds it is the weights' bytes, each loaded once: a wave has two units
// of them (16 rows, 144 or 160 bytes each) in flight, copied into LDS of its
// own as the 16-byte pieces of memory that hold them, wherever in those a
// row begins (loads of each block by a lane of its own, at even addresses 18
// bytes apart, moved 16384 rows of 4096 at 2.7 TB/s, aligned pieces at 5.3).
// Each piece copied holds a byte of the row's, so none is of a page that the
// weights are not in.
// x is copied into LDS before them and split there, a wave taking 512 numbers
// of a row at a time, each such part with a scale of its own and in its own
// place; where x's rows take more than 64 KB, in chunks of K of as many parts
// as fit.  Short calls spend their time on what runs once -- instructions
// fetched, addresses, a barrier -- so little does.
//
// The 16 rows of an MFMA are 4 on each group of lanes, of which a result's 4
// registers are the sums: up to 4 rows of x are one a group, its hi in the
// first register and its lo in the second, up to 8 two a group, so that one
// MFMA takes both parts; from 9 on two do.
//
// Without a chain, in a captured graph: 1 row of 1280 -> 1280 3.9 us (an empty
// launch 1.7); of 4096 -> 16384, Q4_1, 11.1 us, 3.8 TB/s of weights; 2 rows of 1280
// -> 20160 7.4; 33 rows of 2080 -> 1111 8.5; 154 of 768 -> 1280 7.4.
constexpr int kFewWaves = 8;
static_assert(kFewThreads == 64 * kFewWaves);
constexpr int kUnit = 8;        // blocks
// A part of x: 16 blocks of a row, their parts 128 bytes a block (hi, then lo,
// of the four groups), and 16 bytes that spread the rows over the banks.
constexpr int kPart = 16;
constexpr int kPartBytes = 128 * kPart + 16;
constexpr int kFewParts = 32;  // in LDS at a time

// A unit's 16 rows in LDS: at most 11 pieces of 16 bytes each, which also
// spreads the rows over the banks; three copies of 64 pieces bring them, and
// repeat pieces past the last.
constexpr int kPieces = 11;
constexpr int kCopies = 3;
constexpr int kUnitBytes = kCopies * 1024;
constexpr int kRing = 2 * kUnitBytes;  // a wave's

struct FewArgs {
    Q4Args a;
    int32_t splits, tiles;  // S, P
    int32_t ring;           // the waves' rings' place in LDS
    int32_t aligned;        // x begins at a multiple of 16
};

// ROWS of x a workgroup: 1, 2, 4, 8 or 16, the last ones perhaps past M.
template <bool LEAST, bool GATED, int ROWS>
__global__ __launch_bounds__(kFewThreads, 4) void q4_few_kernel(FewArgs f) {
    const Q4Args &a = f.a;
    constexpr int R = ROWS <= 4 ? 1 : ROWS / 4;  // a group's rows
    constexpr int kSize = LEAST ? 20 : 18;
    constexpr bool kJoined = R < 4;  // both parts in one MFMA
    constexpr int kChunk = kFewParts / ROWS * kPart / kUnit;  // units
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ uint32_t exponents[kFewParts];  // of the parts' scales
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, group = lane >> 4;
    const int S = f.splits, P = f.tiles;
    const int split = wave & (S - 1), tile = wave / S, waves = S * P;
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * ROWS;
    const int rows = static_cast<int>(a.M - m0 < ROWS ? a.M - m0 : ROWS);
    const int blocks = static_cast<int>(a.K / kBlock);
    const int units = (blocks + kUnit - 1) / kUnit;
    const int outs = GATED ? P / 2 : P;  // tiles of the output
    const int columns = static_cast<int>(GATED ? a.half : a.N);
    const int n0 = static_cast<int>(blockIdx.x) * (16 * outs);

    // Part u of x's is row u % ROWS's numbers from block u / ROWS * 16 of the
    // chunk on; those past the last block repeat it, those past M its last row.
    const auto fetch_parts = [&](int b0, int count, int share) {
#pragma unroll 1
        for (int u = wave; u < share; u += waves) {
            const int row = u % ROWS;
            const float *x = a.x + (m0 + (row < rows ? row : rows - 1)) * a.ldx + static_cast<int64_t>(b0) * kBlock;
            const int first = u / ROWS * (kPart * kBlock), last = count * kBlock;
            const uint32_t to = lds_address(lds) + kPartBytes * u;
            if (f.aligned) {
                const int at = first + 4 * lane;
                fetch16(x + (at < last ? at : last - 4), to);
                fetch16(x + (at + 256 < last ? at + 256 : last - 4), to + 1024);
            } else {
#pragma unroll 1
                for (int c = 0; c < 8; ++c) {
                    const int at = first + 64 * c + lane;
                    fetch4(x + (at < last ? at : last - 1), to + 256 * c);
                }
            }
        }
    };
    const auto split_parts = [&](int share) {
#pragma unroll 1
        for (int u = wave; u < share; u += waves) {
            // A lane's 8 numbers, 4 group .. and 16 + 4 group .. of a block,
            // make way for their hi and their lo.
            char *place = lds + kPartBytes * u + 128 * (lane >> 2) + 16 * (lane & 3);
            const float4v low = *reinterpret_cast<const float4v *>(place);
            const float4v high = *reinterpret_cast<const float4v *>(place + 64);
            const uint32_t p = magnitude(low), q = magnitude(high);
            const uint32_t e = scale_exponent(wave_greatest(p > q ? p : q));
            half8 hi, lo;
            split8(low, high, power(e), hi, lo);
            *reinterpret_cast<half8 *>(place) = hi;
            *reinterpret_cast<half8 *>(place + 64) = lo;
            if (lane == 0) exponents[u] = e;
        }
    };
    const int count0 = kUnit * kChunk < blocks ? kUnit * kChunk : blocks;
    const int share0 = ROWS * ((count0 + kPart - 1) / kPart);
    fetch_parts(0, count0, share0);

    const auto weights = [&](int c) {  // row c of the wave's tile, or the last there is
        const bool second = GATED && tile >= outs;
        const int n = n0 + 16 * (second ? tile - outs : tile) + c;
        return a.w + ((n < columns ? n : columns - 1) + (second ? columns : 0)) * a.row_bytes;
    };
    const uint8_t *source[kCopies];  // the piece of memory the row of this lane's piece begins in, ...
    int skip[kCopies], piece[kCopies];  // ... how far, and this lane's piece
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
        const int slot = 64 * c + lane, row = slot / kPieces < 16 ? slot / kPieces : 15;
        const uint8_t *at = weights(row);
        skip[c] = static_cast<int>(reinterpret_cast<uintptr_t>(at) & 15);
        source[c] = at - skip[c];
        piece[c] = 16 * (slot - kPieces * row);
    }
    char *ring = lds + f.ring + wave * kRing;
    const auto copy_unit = [&](int u, int buffer) {
        const int count = blocks - kUnit * u < kUnit ? blocks - kUnit * u : kUnit;
#pragma unroll
        for (int c = 0; c < kCopies; ++c) {
            const int last = (skip[c] + kSize * count - 1) & ~15;  // the piece the row's last byte is in
            fetch16(source[c] + u * (kUnit * kSize) + (piece[c] < last ? piece[c] : last),
                    lds_address(ring) + buffer * kUnitBytes + 1024 * c);
        }
    };
    if (split < units) copy_unit(split, 0);
    if (split + S < units) copy_unit(split + S, 1);
    // This lane's row of a unit, and its word of the first block and of the
    // second.  Q4_0's words lie at even addresses, 18 bytes apart, and LDS
    // reads of 4 bytes are fast at multiples of 4 only (16384 rows of 4096:
    // 14.3 us, so 11.9): the two aligned words around one are read and shifted,
    // by nothing or 16 bits, every second block alike.
    const char *mine = ring + 16 * kPieces * col + static_cast<int>(reinterpret_cast<uintptr_t>(weights(col)) & 15);
    const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(mine + kSize - 16) & 2);  // the first's
    const char *words[2] = {mine + kSize - 16 + 4 * group - odd, mine + 2 * kSize - 16 + 4 * group - (LEAST ? odd : 2 - odd)};
    const uint32_t shift[2] = {8u * odd, LEAST ? 8u * odd : 16u - 8u * odd};
    // The row of x that this lane's row of the MFMA is, and its part.
    const int token = (R == 1 ? col >> 2 : R == 2 ? col >> 1 : col) & (ROWS - 1);
    const char *numbers = lds + kPartBytes * token + (kJoined ? 64 * (col & 1) : 0) + 16 * group;
    // x's parts are in: a wave's loads end in order.
    if (split + S < units) {
        fetched<2 * kCopies>();
    } else if (split < units) {
        fetched<kCopies>();
    } else {
        fetched<0>();
    }
    split_parts(share0);
    float sum[R];
#pragma unroll
    for (int e = 0; e < R; ++e) sum[e] = 0.0f;
    const uint32_t magic = opaque(kMagic);
    int buffer = 0;
    for (int u0 = 0;;) {
        const int u1 = u0 + kChunk < units ? u0 + kChunk : units;
        lds_barrier();
#pragma unroll 1
        for (int u = u0 + split; u < u1; u += S) {
            // This unit's copies are in; those of the one after may not be.
            if (u + S < units) {
                fetched<kCopies>();
            } else {
                fetched<0>();
            }
            const int part = (u - u0) / (kPart / kUnit) * ROWS;
            const char *row = mine + buffer * kUnitBytes;
            const char *x = numbers + kPartBytes * part + (u - u0) % (kPart / kUnit) * (128 * kUnit);
            float acc[R];
#pragma unroll
            for (int e = 0; e < R; ++e) acc[e] = 0.0f;
            const auto add_block = [&](int i, int odd_block) {
                const char *block = row + kSize * i;
                const uint32_t *at = reinterpret_cast<const uint32_t *>(words[odd_block] + buffer * kUnitBytes +
                                                                        kSize * (i - odd_block));
                const uint32_t word = __builtin_amdgcn_alignbit(at[1], at[0], shift[odd_block]);
                _Float16 d;
                __builtin_memcpy(&d, block, 2);
                const half8 x0 = *reinterpret_cast<const half8 *>(x + 128 * i);
                half8 x1;
                if constexpr (!kJoined) x1 = *reinterpret_cast<const half8 *>(x + 128 * i + 64);
                const auto times = [&](const half8 &v, float (&p)[R]) {
                    const float4v zero = {0.0f, 0.0f, 0.0f, 0.0f};
                    float4v r;
                    if constexpr (kJoined) {
                        r = __builtin_amdgcn_mfma_f32_16x16x32_f16(x0, v, zero, 0, 0, 0);
#pragma unroll
                        for (int e = 0; e < R; ++e) p[e] = r[2 * e] + r[2 * e + 1];
                    } else {
                        r = __builtin_amdgcn_mfma_f32_16x16x32_f16(x1, v, zero, 0, 0, 0);
                        r = __builtin_amdgcn_mfma_f32_16x16x32_f16(x0, v, r, 0, 0, 0);
#pragma unroll
                        for (int e = 0; e < R; ++e) p[e] = r[e];
                    }
                };
                float p[R];
                times(widen(word, magic), p);
                const float scale = static_cast<float>(d);
#pragma unroll
                for (int e = 0; e < R; ++e) acc[e] = __builtin_fmaf(scale, p[e], acc[e]);
                if constexpr (LEAST) {
                    _Float16 least;
                    __builtin_memcpy(&least, block + 2, 2);
                    times(half8{1, 1, 1, 1, 1, 1, 1, 1}, p);
                    const float offset = __builtin_fmaf(8.0f, scale, static_cast<float>(least));
#pragma unroll
                    for (int e = 0; e < R; ++e) acc[e] = __builtin_fmaf(offset, p[e], acc[e]);
                }
            };
            const int count = blocks - kUnit * u < kUnit ? blocks - kUnit * u : kUnit;
            int i = 0;
#pragma unroll 1
            for (; i + 4 <= count; i += 4) {
#pragma unroll
                for (int j = 0; j < 4; ++j) add_block(i + j, j & 1);
            }
#pragma unroll 1
            for (; i < count; ++i) add_block(i, i & 1);
            // The scale of its part out of the unit's sums.
#pragma unroll
            for (int e = 0; e < R; ++e) {
                const uint32_t back = 254 - exponents[part + ((R * group + e) & (ROWS - 1))];
                sum[e] = __builtin_fmaf(acc[e], power(back), sum[e]);
            }
            if (u + 2 * S < units) {
                // The unit is read: the one two on takes its place.
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
                copy_unit(u + 2 * S, buffer);
            }
            buffer ^= 1;
        }
        lds_barrier();  // the chunk's parts read
        u0 = u1;
        if (u0 == units) break;
        const int b0 = kUnit * u0, left = blocks - b0;
        const int count = kUnit * kChunk < left ? kUnit * kChunk : left;
        const int share = ROWS * ((count + kPart - 1) / kPart);
        fetch_parts(b0, count, share);
        fetched<0>();
        split_parts(share);
    }
    float *sums = reinterpret_cast<float *>(lds);  // [split][tile][register][lane]
#pragma unroll
    for (int e = 0; e < R; ++e) sums[((split * P + tile) * R + e) * 64 + lane] = sum[e];
    lds_barrier();
    const auto place = [&](int at, int64_t &m, int &out) {
        const int row = R * ((at & 63) >> 4) + (at >> 6) % R;
        m = row < rows ? m0 + row : a.M;
        out = n0 + 16 * (at / (64 * R)) + (at & 15);
        return 1.0f;
    };
    if (outs * R * 64 <= 64 * waves) {
        write_outputs<GATED, 1>(a, sums, S, P * R * 64, outs * R * 64, tid, columns, place, 64 * waves);
    } else {
        write_outputs<GATED, R>(a, sums, S, P * R * 64, outs * R * 64, tid, columns, place, 64 * waves);
    }
}

// Rows a workgroup and splits of K: those of the least time, in us.  Beyond
// 2.5 us that a call takes anyhow workgroups that share a CU add up: a part of x
// 0.08, a unit of a wave's weights 0.8 (1.28 where its MFMAs are two), and a
// start of 1.04 for every two that fit its LDS at once, or one (within 7 % of
// what 630 calls of 1 .. 154 rows took, 320 -> 320 to 4096 -> 16384; the choices
// by it 0.2 % slower than the fastest of all).  With 16 rows throughout, 33 rows
// of 2080 -> 1111 took 12.8 us, now 8.8; 16 of 1280 -> 10240 16.6, now 9.9; 24 of
// 768 -> 1280 6.8, now 5.0.  With 8 at most, 256 of 1280 -> 1280 18.7, now 14.6.
// Where the workgroups leave CUs without one, they take as few tiles as fit the
// device, if a wave splits no more than one and a half parts of x then (320 -> 320
// with a bias 4.4 us, so 3.9; 2 rows of 1280 -> 20160 8.2 and 7.9).
struct FewShape {
    int rows, splits, tiles;
    float time;
};

FewShape few_shape(int64_t M, int64_t N, int64_t K, bool gated) {
    constexpr int64_t kLdsBytes = 160 * 1024;
    const auto shifted = [](int64_t v, int by) { return (v + (int64_t{1} << by) - 1) >> by; };  // v / 2^by, rounded up
    const int64_t cus = compute_units(), tiles = ceil_div(N, 16), units = ceil_div(K / kBlock, kUnit);
    FewShape best{0, 0, 0, 0.0f};
    int64_t least = 0;
    for (int r = 0; r <= 4; ++r) {
        const int64_t groups = shifted(M, r), parts = ceil_div(K / kBlock, kPart) << r;
        const int64_t chunk = (kFewParts >> r) * (kPart / kUnit);
        const bool two = 2 * ((parts < kFewParts ? parts : kFewParts) * kPartBytes + kFewWaves * kRing) <= kLdsBytes;
        for (int s = 0; groups <= 65535 && s <= (gated ? 2 : 3); ++s) {
            if (s > 0 && ((1 << (s - 1)) >= units || (1 << s) > chunk)) break;
            const int64_t each = ceil_div(groups * ceil_div(tiles << s, kFewWaves), cus);  // a CU's workgroups
            // In 0.08 us.
            const int64_t cost = each * (shifted(units, s) * (r < 4 ? 10 : 16) + parts) + (two ? shifted(each, 1) : each) * 13;
            if (best.rows == 0 || cost < least) {
                best = {1 << r, 1 << s, kFewWaves >> s, 2.5f + 0.08f * static_cast<float>(cost)};
                least = cost;
            }
        }
        if ((1 << r) >= M) break;
    }
    if (best.rows != 0 && ceil_div(M, best.rows) < cus) {
        const int64_t groups = ceil_div(M, best.rows), parts = ceil_div(K / kBlock, kPart) * best.rows;
        const int64_t fit = ceil_div(tiles, cus / groups), least_tiles = gated ? round_up(fit, 2) : fit;
        if (least_tiles < best.tiles && 2 * parts <= 3 * least_tiles * best.splits) best.tiles = static_cast<int>(least_tiles);
    }
    return best;
}

template <bool LEAST, bool GATED, int ROWS>
hipError_t launch_few(const Q4Args &a, const FewShape &shape, hipStream_t stream) {
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&q4_few_kernel<LEAST, GATED, ROWS>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize,
                                                       kFewParts * kPartBytes + kFewWaves * kRing);
    if (attr != hipSuccess) return attr;
    FewArgs f{};
    f.a = a;
    f.splits = shape.splits;
    const int64_t columns = GATED ? a.half : a.N;
    const int64_t parts = ceil_div(a.K / kBlock, kPart) * ROWS;
    f.tiles = shape.tiles;
    const int waves = f.tiles * f.splits;
    const dim3 grid(static_cast<uint32_t>(ceil_div(columns, 16 * (GATED ? f.tiles / 2 : f.tiles))),
                    static_cast<uint32_t>(ceil_div(a.M, ROWS)));
    f.ring = static_cast<int32_t>(kPartBytes * (parts < kFewParts ? parts : kFewParts));
    f.aligned = reinterpret_cast<uintptr_t>(a.x) % 16 == 0;
    SDHIP_LAUNCH((q4_few_kernel<LEAST, GATED, ROWS>), grid, dim3(64 * waves),
                 static_cast<uint32_t>(f.ring + waves * kRing), stream, f);
    return hipGetLastError();
}

template <bool LEAST, bool GATED>
hipError_t few_rows(const Q4Args &a, hipStream_t stream) {
    const FewShape shape = few_shape(a.M, a.N, a.K, GATED);
    switch (shape.rows) {
    case 1:
        return launch_few<LEAST, GATED, 1>(a, shape, stream);
    case 2:
        return launch_few<LEAST, GATED, 2>(a, shape, stream);
    case 4:
        return launch_few<LEAST, GATED, 4>(a, shape, stream);
    case 8:
        return launch_few<LEAST, GATED, 8>(a, shape, stream);
    default:
        return launch_few<LEAST, GATED, 16>(a, shape, stream);
    }
}

// ------------------------------------------------------------------ many rows

// More rows of x: both operands are first laid out in the work buffer as the
// products' lanes read them (q4_operands_kernel), then multiplied by tiles
// (q4_tiles_kernel).
//
// x: for every block and 32 rows 4 KB, [16 numbers' half of the block][hi, lo]
// [lane][8], lane 32 h + row holding the block's word 2 half + h of its row, the
// 8 numbers in widen's order; a row has one scale, from its greatest number.
// The weights: for every block and 32 rows of them 640 bytes, the two words
// of lane 32 h + row side by side, then the 32 rows' d in single precision.  For
// the gated product 32 rows of each half of the weights take turns.
//
// Q4_1's offsets c times the blocks' sums of x are a product of their own, 32
// blocks its step, of three bfloat16 parts each (24 bits of any magnitude): six
// MFMAs for what would be 32 multiplications and additions an output.  Both
// lie as the MFMA reads them, 6 KB a 32 rows and 32 blocks: [16 blocks][part]
// [lane 32 h + row][8 blocks].
constexpr int kRowsTile = 32;
constexpr int64_t kNumbersBytes = 4096, kWordsBytes = 640, kOffsetsBytes = 6144;

struct TileArgs {
    Q4Args a;
    char *numbers, *words;  // x's parts; the weights' words and scales
    float *back;            // a row of x's scale out of its sums
    char *sums, *offsets;   // Q4_1: the blocks' sums of x; c
    int32_t blocks, groups;  // of 32 numbers; of 32 blocks
    int32_t row_tiles, column_tiles;  // 32 rows each, whole workgroups' of them
    int32_t x_groups;       // workgroups that lay x out
    int32_t m_blocks, n_blocks;
};

// v in three bfloat16 parts, each what the ones before leave.
__device__ __forceinline__ void split_bf16(float v, __bf16 (&p)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        p[i] = static_cast<__bf16>(v);
        // An infinity is all in the first.
        v = __builtin_isinf(v) ? 0.0f : v - static_cast<float>(p[i]);
    }
}

constexpr int kOperandThreads = 512;
constexpr int kOperandRows = 8;  // of x a workgroup

// Workgroups of two kinds: 8 rows of x, or 32 rows of the weights by 32 blocks.
// A wave takes 2 blocks of the 8 rows at a time, 8 lanes a row, so that what it
// reads of a row lies together and what it writes of them does too; the first
// kKept such times are kept in registers while the rows' greatest are found
// (1976 rows of 5120: 30 us with a row a wave, written 16 bytes here and there, now
// 18.5, 5.9 TB/s).
template <bool LEAST, bool GATED>
__global__ __launch_bounds__(kOperandThreads) void q4_operands_kernel(TileArgs t) {
    const Q4Args &a = t.a;
    constexpr int kSize = LEAST ? 20 : 18;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (static_cast<int>(blockIdx.x) < t.x_groups) {
        constexpr int kWaves = kOperandThreads / 64, kKept = 6;
        __shared__ uint32_t greatest[kWaves][kOperandRows];
        const int64_t m = static_cast<int64_t>(blockIdx.x) * kOperandRows + (lane >> 3);
        const int word = lane & 3, first = 2 * wave + ((lane >> 2) & 1);
        const float *x = a.x + (m < a.M ? m : a.M - 1) * a.ldx + 4 * word;
        const auto load = [&](int b, float4v &low, float4v &high) {
            low = float4v{0.0f, 0.0f, 0.0f, 0.0f};
            high = low;
            if (b < t.blocks) {
                low = load4(x + b * static_cast<int64_t>(kBlock));
                high = load4(x + b * static_cast<int64_t>(kBlock) + 16);
            }
        };
        const auto greater = [](uint32_t p, uint32_t q) { return p > q ? p : q; };
        float4v low[kKept], high[kKept];
#pragma unroll
        for (int i = 0; i < kKept; ++i) load(first + 2 * kWaves * i, low[i], high[i]);
        uint32_t v = 0;
#pragma unroll
        for (int i = 0; i < kKept; ++i) v = greater(v, greater(magnitude(low[i]), magnitude(high[i])));
        for (int b = first + 2 * kWaves * kKept; b < t.blocks; b += 2 * kWaves) {
            float4v l, h;
            load(b, l, h);
            v = greater(v, greater(magnitude(l), magnitude(h)));
        }
        v = greater(v, __builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, true));   // lanes i ^ 1
        v = greater(v, __builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, true));   // i ^ 2
        v = greater(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true));  // 8 lanes mirrored
        if ((lane & 7) == 0) greatest[wave][lane >> 3] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) v = greater(v, greatest[w][lane >> 3]);
        const uint32_t e = scale_exponent(v);
        const float scale = power(e);
        if (m < a.M && wave == 0 && (lane & 7) == 0) t.back[m] = power(254 - e);
        const int64_t tile = m / kRowsTile;
        const int row = static_cast<int>(m % kRowsTile);
        const auto write = [&](int b, const float4v &l, const float4v &h) {
            float sum = 0.0f;
            if (b < t.blocks && m < a.M) {
                half8 hi, lo;
                split8(l, h, scale, hi, lo);
                char *to = t.numbers + (b * static_cast<int64_t>(t.row_tiles) + tile) * kNumbersBytes + (word >> 1) * 2048 +
                           ((word & 1) * 32 + row) * 16;
                *reinterpret_cast<half8 *>(to) = hi;
                *reinterpret_cast<half8 *>(to + 1024) = lo;
                if constexpr (LEAST) {
                    // Scaled before they are added: sums of x itself may pass single precision.
                    const float4v p = l * scale, q = h * scale;
                    sum = ((p[0] + p[1]) + (p[2] + p[3])) + ((q[0] + q[1]) + (q[2] + q[3]));
                }
            }
            if constexpr (LEAST) {
                sum += __shfl_xor(sum, 1, 64);
                sum += __shfl_xor(sum, 2, 64);
                if (word == 0 && m < a.M && b < t.groups * 32) {
                    __bf16 p[3];
                    split_bf16(sum, p);
                    char *to = t.sums + ((b >> 5) * static_cast<int64_t>(t.row_tiles) + tile) * kOffsetsBytes +
                               ((b >> 4) & 1) * 3072 + (((b >> 3) & 1) * 32 + row) * 16 + 2 * (b & 7);
#pragma unroll
                    for (int i = 0; i < 3; ++i) *reinterpret_cast<__bf16 *>(to + 1024 * i) = p[i];
                }
            }
        };
#pragma unroll
        for (int i = 0; i < kKept; ++i) write(first + 2 * kWaves * i, low[i], high[i]);
        // Q4_1: the sums of the blocks that fill the last 32 are 0.
        for (int b = first + 2 * kWaves * kKept; b < (LEAST ? t.groups * 32 : t.blocks); b += 2 * kWaves) {
            float4v l, h;
            load(b, l, h);
            write(b, l, h);
        }
        return;
    }
    // Strips of 16 blocks, one for each half of the workgroup.  Rows of pieces
    // that hold 16 blocks wherever they begin, an odd number of them to spread
    // the rows over the banks.
    constexpr int kRow = LEAST ? 21 : 19;
    constexpr int kHalf = kOperandThreads / 2;
    constexpr int kRounds = (kRowsTile * kRow + kHalf - 1) / kHalf;
    __shared__ __attribute__((aligned(16))) char lds[2][kRounds * kHalf * 16];
    const int pairs = LEAST ? t.groups : (t.blocks + 31) / 32;
    const int item = static_cast<int>(blockIdx.x) - t.x_groups;
    const int half = wave / (kHalf / 64), place = tid & (kHalf - 1);
    const int tile = item / pairs, b0 = (item % pairs * 2 + half) * 16;
    const int count = t.blocks - b0 < 16 ? t.blocks - b0 : 16;  // 0 and less: zeros of offsets only
    const auto weights = [&](int r) {
        const int64_t columns = GATED ? a.half : a.N;
        const int64_t n = (GATED ? tile >> 1 : tile) * kRowsTile + r;
        return a.w + ((n < columns ? n : columns - 1) + (GATED && (tile & 1) ? a.half : 0)) * a.row_bytes + b0 * kSize;
    };
    if (count > 0) {
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            const int slot = kHalf * i + place;
            const int row = slot / kRow < kRowsTile ? slot / kRow : kRowsTile - 1;
            const uint8_t *at = weights(row);
            const int skip = static_cast<int>(reinterpret_cast<uintptr_t>(at) & 15);
            const int piece = 16 * (slot - kRow * row), last = (skip + kSize * count - 1) & ~15;
            fetch16(at - skip + (piece < last ? piece : last),
                    lds_address(lds[half]) + kHalf * 16 * i + 1024 * (wave & (kHalf / 64 - 1)));
        }
        fetched<0>();
    }
    lds_barrier();
    const int col = lane & 31, h = lane >> 5;
    const char *mine = lds[half] + 16 * kRow * col + static_cast<int>(reinterpret_cast<uintptr_t>(weights(col)) & 15);
    for (int i = wave & (kHalf / 64 - 1); i < count; i += kHalf / 64) {
        const char *block = mine + kSize * i;
        uint32_t w[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) __builtin_memcpy(&w[s], block + kSize - 16 + 8 * s + 4 * h, 4);
        _Float16 d;
        __builtin_memcpy(&d, block, 2);
        char *to = t.words + ((b0 + i) * static_cast<int64_t>(t.column_tiles) + tile) * kWordsBytes;
        *reinterpret_cast<uint2 *>(to + 8 * lane) = make_uint2(w[0], w[1]);
        if (h == 0) *reinterpret_cast<float *>(to + 512 + 4 * col) = static_cast<float>(d);
    }
    if constexpr (LEAST) {
        if ((wave & (kHalf / 64 - 1)) == 0) {
            // Lane 32 h + row: the offsets of the strip's blocks 8 h .. 8 h + 7.
            typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
            bf16x8 p[3];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int i = 8 * h + j;
                float c = 0.0f;
                if (i < count) {
                    _Float16 d, least;
                    __builtin_memcpy(&d, mine + kSize * i, 2);
                    __builtin_memcpy(&least, mine + kSize * i + 2, 2);
                    c = __builtin_fmaf(8.0f, static_cast<float>(d), static_cast<float>(least));
                }
                __bf16 q[3];
                split_bf16(c, q);
#pragma unroll
                for (int k = 0; k < 3; ++k) p[k][j] = q[k];
            }
            char *to = t.offsets + ((b0 >> 5) * static_cast<int64_t>(t.column_tiles) + tile) * kOffsetsBytes +
                       ((b0 >> 4) & 1) * 3072 + 16 * lane;
#pragma unroll
            for (int k = 0; k < 3; ++k) *reinterpret_cast<bf16x8 *>(to + 1024 * k) = p[k];
        }
    }
}

// Tiles of 64 WM rows of x by 32 TN WN of the weights, a wave 64 x 32 TN of them
// and one block of every WK: 8 TN v_mfma_f32_32x32x16_f16 a block.  The operands of
// WK blocks come into LDS in runs, three stages of them in turn, asked for two
// stages ahead.  With TN 2 a block's sums of products are scaled by d, 64
// operations beside the 36 that widen the words, 400 of the vector units' cycles
// a block to 512 of the MFMA's.  No one unit bounds it: 1976 rows of 1280 -> 2 x
// 5120 gated take 126 us, the MFMA busy 44 % of the cycles at the 1.9 GHz that
// this product runs at; without any one of the copies, the scaling, the widening
// or the barriers 116 .. 127, without the reads of LDS 98.
template <int WM, int WN, int WK, int TN>
struct Tiles {
    static constexpr int kWaves = WM * WN * WK;
    static constexpr int kThreads = 64 * kWaves;
    static constexpr int kNumbers = WM * 2 * 4;                   // KB a block
    static constexpr int kWords = (WN * TN * kWordsBytes + 1023) / 1024;  // KB a block, rounded up
    static constexpr int kPerBlock = kNumbers + kWords;
    static constexpr int kCopies = (WK * kPerBlock + kWaves - 1) / kWaves;  // a wave's, a stage
    static constexpr int kStage = kCopies * kWaves * 1024;
    static constexpr int kStages = 3;
    static constexpr int kJoined = TN % 2 == 0 ? 2 : 1;  // of the TN whose sums the waves of WK blocks add up at a time
    static constexpr int kSums = WK > 1 ? kWaves * kJoined * 8192 : 0;
    static constexpr int kLds = kStages * kStage > kSums ? kStages * kStage : kSums;
};

// The order of what was written since the last sched_barrier: four MFMAs, N
// vector operations after each.
template <int N>
__device__ __forceinline__ void mixed() {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, N, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
}

template <bool LEAST, bool GATED, int WM, int WN, int WK, int TN>
__global__ __launch_bounds__(64 * WM * WN * WK, 2) void q4_tiles_kernel(TileArgs t) {
    using L = Tiles<WM, WN, WK, TN>;
    const Q4Args &a = t.a;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wk = wave % WK, wn = wave / WK % WN, wm = wave / (WK * WN);
    const uint32_t at = xcd_swizzle(blockIdx.x, gridDim.x);
    const int mb = at / t.n_blocks, nb = at - mb * t.n_blocks;
    const int stages = (t.blocks + WK - 1) / WK;
    // A wave's copies of a stage: kCopies KB of its WK kPerBlock, the last ones
    // perhaps again.  A block past the last is the last.
    const char *from[L::kCopies];
    int64_t step[L::kCopies];
    int block[L::kCopies];
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_address(lds) + 1024 * wave * L::kCopies);
#pragma unroll
    for (int c = 0; c < L::kCopies; ++c) {
        int q = wave * L::kCopies + c;
        q = q < WK * L::kPerBlock ? q : WK * L::kPerBlock - 1;
        const int r = q % L::kPerBlock;
        block[c] = q / L::kPerBlock;
        from[c] = r < L::kNumbers ? t.numbers + mb * (WM * 2) * kNumbersBytes + 1024 * r
                                  : t.words + nb * (WN * TN) * kWordsBytes + 1024 * (r - L::kNumbers);
        step[c] = r < L::kNumbers ? t.row_tiles * kNumbersBytes : t.column_tiles * kWordsBytes;
    }
    const auto copy = [&](int s, int buffer, int c) {
        const int b = s * WK + block[c] < t.blocks ? s * WK + block[c] : t.blocks - 1;
        fetch16(from[c] + b * step[c], 16 * lane, to + buffer * L::kStage + 1024 * c);
    };
#pragma unroll
    for (int s = 0; s < 3; ++s)
#pragma unroll
        for (int c = 0; c < L::kCopies; ++c) copy(s, s, c);
    float16v acc[2][TN];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = float16v{};
    const uint32_t magic = opaque(kMagic);
    const char *x = lds + wk * (L::kPerBlock * 1024) + wm * 8192 + 16 * lane;
    const char *w = lds + wk * (L::kPerBlock * 1024) + L::kNumbers * 1024 + wn * TN * static_cast<int>(kWordsBytes);
    struct Operands {
        half8 n[2][2][2];  // [32 rows][half of the block][hi, lo]
        half8 v[TN][2];    // [32 rows of the weights][half of the block]
        uint2 words[TN];   // v before it is widened
        float d[TN];
    };
    const auto read = [&](Operands &o, int buffer) {
        const char *xs = x + buffer * L::kStage, *ws = w + buffer * L::kStage;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int p = 0; p < 4; ++p) o.n[i][p >> 1][p & 1] = *reinterpret_cast<const half8 *>(xs + 4096 * i + 1024 * p);
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            o.words[j] = *reinterpret_cast<const uint2 *>(ws + kWordsBytes * j + 8 * lane);
            o.d[j] = *reinterpret_cast<const float *>(ws + kWordsBytes * j + 512 + 4 * (lane & 31));
        }
    };
    const auto widen_words = [&](Operands &o, int j) {
        o.v[j][0] = widen(o.words[j].x, magic);
        o.v[j][1] = widen(o.words[j].y, magic);
    };
    const auto product = [&](const Operands &o, int i, int j) {
        float16v p = __builtin_amdgcn_mfma_f32_32x32x16_f16(o.n[i][0][1], o.v[j][0], float16v{}, 0, 0, 0);
        p = __builtin_amdgcn_mfma_f32_32x32x16_f16(o.n[i][1][1], o.v[j][1], p, 0, 0, 0);
        p = __builtin_amdgcn_mfma_f32_32x32x16_f16(o.n[i][0][0], o.v[j][0], p, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(o.n[i][1][0], o.v[j][1], p, 0, 0, 0);
    };
    const auto add = [&](int i, int j, float d, const float16v &p) {
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = __builtin_fmaf(d, p[e], acc[i][j][e]);
    };
    // A block's products; a product's sums are added up while the MFMA makes the
    // next one's, the last's in the next block.
    float16v kept = float16v{};
    float kept_d = 0.0f;
    const auto multiply = [&](const Operands &o, auto between) {
        __builtin_amdgcn_sched_barrier(0);
        float16v p = kept;
        float d = kept_d;
        int i = 1, j = TN - 1;
#pragma unroll
        for (int k = 0; k < 2 * TN; ++k) {
            const float16v next = product(o, k & 1, k >> 1);
            between(k);
            add(i, j, d, p);
            p = next;
            i = k & 1;
            j = k >> 1;
            d = o.d[j];
            if (k < TN) {
                mixed<4>();
            } else {
                mixed<9>();
            }
        }
        kept = p;
        kept_d = d;
    };
    fetched<2 * L::kCopies>();
    lds_barrier();
    Operands even, odd;
    read(even, 0);
#pragma unroll
    for (int j = 0; j < TN; ++j) widen_words(even, j);
    int buffer = 0;
    // Stage s is multiplied from registers while stage s + 1 is read into
    // others; s + 2 is under way and s + 3 takes the buffer that s was read
    // from -- for the last stages, the last one again.
    const auto stage = [&](int s, const Operands &now, Operands &next) {
        fetched<L::kCopies>();
        lds_barrier();  // every wave's copies of stage s + 1 are in, and stage s is read
        const int free = buffer;
        buffer = buffer == 2 ? 0 : buffer + 1;
        multiply(now, [&](int k) {
            if (k == 0) read(next, buffer);
            if (k >= TN) widen_words(next, k - TN);
#pragma unroll
            for (int c = 0; c < L::kCopies; ++c)
                if (c * 2 * TN / L::kCopies == k) copy(s + 3, free, c);
        });
    };
    int s = 0;
#pragma unroll 1
    for (; s + 2 < stages; s += 2) {
        stage(s, even, odd);
        stage(s + 1, odd, even);
    }
    if (s + 1 < stages) {
        stage(s, even, odd);
        even = odd;
        ++s;
    }
    if (s * WK + wk < t.blocks) multiply(even, [](int) {});
    add(1, TN - 1, kept_d, kept);
    fetched<0>();
    if constexpr (LEAST) {
        typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
        struct Parts {
            bf16x8 u[2][3], v[TN][3];
        };
        // Step k: 16 blocks, half k % 2 of the wave's group k / 2.
        const int steps = wk < t.groups ? 2 * ((t.groups - wk + WK - 1) / WK) : 0;
        const auto load = [&](int k, Parts &o) {
            const int64_t g = wk + (k >> 1) * WK;
            const char *sums = t.sums + (g * t.row_tiles + mb * (WM * 2) + wm * 2) * kOffsetsBytes + 3072 * (k & 1) + 16 * lane;
            const char *offs = t.offsets + (g * t.column_tiles + nb * (WN * TN) + wn * TN) * kOffsetsBytes + 3072 * (k & 1) + 16 * lane;
#pragma unroll
            for (int p = 0; p < 3; ++p) {
#pragma unroll
                for (int i = 0; i < 2; ++i) o.u[i][p] = *reinterpret_cast<const bf16x8 *>(sums + i * kOffsetsBytes + 1024 * p);
#pragma unroll
                for (int j = 0; j < TN; ++j) o.v[j][p] = *reinterpret_cast<const bf16x8 *>(offs + j * kOffsetsBytes + 1024 * p);
            }
        };
        // The parts' products down to 2^-16 of the whole, the least first.
        const auto multiply_parts = [&](const Parts &o) {
#pragma unroll
            for (int total = 2; total >= 0; --total)
#pragma unroll
                for (int p = 0; p <= total; ++p)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int j = 0; j < TN; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(o.u[i][p], o.v[j][total - p], acc[i][j], 0, 0, 0);
        };
        Parts a0, a1;
        if (steps > 0) load(0, a0);
#pragma unroll 1
        for (int k = 0; k < steps; k += 2) {
            load(k + 1, a1);
            multiply_parts(a0);
            if (k + 2 < steps) load(k + 2, a0);
            multiply_parts(a1);
        }
    }
    // The outputs by quarters of the wave's, 8 rows a lane of kJoined of its
    // columns: rows 16 (q % 2) .. of its 32 q / 2.  The waves of WK blocks add up
    // a part of the quarters each; a wave alone takes one or two at a time.
    constexpr int J = L::kJoined;
    constexpr int kQuarters = WK == 4 || (WK == 1 && GATED) ? 1 : 2;
    constexpr int kWaveSums = J * 2048;  // floats
    static_assert(!GATED || TN == 2);
    const float *all = reinterpret_cast<const float *>(lds) + (wave - wk) * kWaveSums + lane;
    const int64_t columns = GATED ? a.half : a.N;
    const int m0 = mb * (64 * WM) + wm * 64 + 4 * (lane >> 5);
    const int first = (nb * WN + wn) * (GATED ? 32 : 32 * TN) + (lane & 31);
#pragma unroll
    for (int round = 0; round < TN / J * (4 / WK / kQuarters); ++round) {
        const int j0 = WK == 1 ? 0 : J * round, n0 = first + 32 * j0;
        if constexpr (WK > 1) {
            lds_barrier();  // the last stage is read, and no copy is under way; the sums before are
            float *sums = reinterpret_cast<float *>(lds) + wave * kWaveSums + lane;  // [quarter][j][e][lane]
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) sums[((q * J + j) * 8 + e) * 64] = acc[q >> 1][j0 + j][8 * (q & 1) + e];
            lds_barrier();
        }
        const int q0 = WK == 1 ? kQuarters * round : wk * kQuarters;
        float v[kQuarters][J][8];
#pragma unroll
        for (int q = 0; q < kQuarters; ++q)
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if constexpr (WK == 1) {
                        v[q][j][e] = acc[(kQuarters * round + q) >> 1][j][8 * ((kQuarters * round + q) & 1) + e];
                    } else {
                        v[q][j][e] = 0.0f;
#pragma unroll
                        for (int k = 0; k < WK; ++k) v[q][j][e] += all[k * kWaveSums + (((q0 + q) * J + j) * 8 + e) * 64];
                    }
                }
        const auto row_of = [&](int q, int e) { return m0 + 16 * (q0 + q) + tile_row(e); };
        const auto column_of = [&](int j) -> int64_t {  // j's column, or the last there is
            const int64_t n = GATED ? n0 : n0 + 32 * j;
            return (n < columns ? n : columns - 1) + (GATED && j ? a.half : 0);
        };
        const int64_t last = a.M - 1;
#pragma unroll
        for (int q = 0; q < kQuarters; ++q)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float back = t.back[row_of(q, e)];
#pragma unroll
                for (int j = 0; j < J; ++j) v[q][j][e] *= back;
            }
        if (!GATED && a.from_redirect) {
#pragma unroll
            for (int q = 0; q < kQuarters; ++q)
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int64_t m = row_of(q, e) < last ? row_of(q, e) : last;
                        v[q][j][e] = a.y[m * a.ldy + column_of(j)] + v[q][j][e];
                    }
        }
        // The chain, a step's operands all asked for before one is used.
#pragma unroll 1
        for (int c = 0; c < a.chain.count; ++c) {
            const DevStep &st = a.chain.steps[c];
            if (st.kind == kSilu) {
#pragma unroll
                for (int q = 0; q < kQuarters; ++q)
#pragma unroll
                    for (int j = 0; j < J; ++j)
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[q][j][e] = silu(v[q][j][e]);
                continue;
            }
            float o[kQuarters][J][8];
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const float *at = st.operand + column_of(j) * st.nb[0];
                if (st.flat123 && st.nb[1] == 0) {
                    const float one = *at;
#pragma unroll
                    for (int q = 0; q < kQuarters; ++q)
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[q][j][e] = one;
                } else if (st.flat123) {
#pragma unroll
                    for (int q = 0; q < kQuarters; ++q)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            o[q][j][e] = at[(row_of(q, e) < last ? row_of(q, e) : last) * st.nb[1]];
                } else {
#pragma unroll
                    for (int q = 0; q < kQuarters; ++q)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int64_t m = row_of(q, e) < last ? row_of(q, e) : last;
                            uint32_t i1, i2, i3;
                            split_index(static_cast<uint32_t>(m), static_cast<uint32_t>(a.ne1), static_cast<uint32_t>(a.ne2),
                                        i1, i2, i3);
                            o[q][j][e] = at[i1 * st.nb[1] + i2 * st.nb[2] + i3 * st.nb[3]];
                        }
                }
            }
#pragma unroll
            for (int q = 0; q < kQuarters; ++q)
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        v[q][j][e] = st.kind == kAdd ? __fadd_rn(v[q][j][e], o[q][j][e]) : __fmul_rn(v[q][j][e], o[q][j][e]);
        }
#pragma unroll
        for (int q = 0; q < kQuarters; ++q)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int64_t m = row_of(q, e);
                if (m > last) continue;
                float *y = a.y + m * a.ldy;
                if constexpr (GATED) {
                    if (n0 < columns) y[n0] = v[q][0][e] * gelu(v[q][1][e]);
                } else {
#pragma unroll
                    for (int j = 0; j < J; ++j)
                        if (n0 + 32 * j < columns) y[n0 + 32 * j] = v[q][j][e];
                }
            }
    }
}

template <bool LEAST, bool GATED, int WM, int WN, int WK, int TN>
hipError_t launch_tiles(TileArgs t, hipStream_t stream) {
    using L = Tiles<WM, WN, WK, TN>;
    static const hipError_t attr =
        hipFuncSetAttribute(reinterpret_cast<const void *>(&q4_tiles_kernel<LEAST, GATED, WM, WN, WK, TN>),
                            hipFuncAttributeMaxDynamicSharedMemorySize, L::kLds);
    if (attr != hipSuccess) return attr;
    t.m_blocks = static_cast<int32_t>(ceil_div(t.a.M, 64 * WM));
    t.n_blocks = static_cast<int32_t>(GATED ? ceil_div(t.a.half, 32 * WN) : ceil_div(t.a.N, 32 * TN * WN));
    SDHIP_LAUNCH((q4_tiles_kernel<LEAST, GATED, WM, WN, WK, TN>), dim3(static_cast<uint32_t>(t.m_blocks * t.n_blocks)),
                 dim3(L::kThreads), L::kLds, stream, t);
    return hipGetLastError();
}

// ------------------------------------------------------------------ rows between

// Rows of x too many to split in every workgroup and too few for tiles: x is
// laid out as for the tiles, the weights are read as they are.  A workgroup
// takes P tiles of 32 rows of the weights by S splits of K, a wave each, and
// 32 MT rows of x; a wave's weights come into LDS of its own by units of 8
// blocks, two of them in flight, as few rows' do, and x from L2 as the MFMA's
// lanes want it, a block ahead.  Q4_1's offsets go by bfloat16 parts as the
// tiles' do, a unit's 8 blocks one step of v_mfma_f32_32x32x8_bf16.  Bound by x's
// loads from L2, 4 KB a wave, block and 32 rows (256 rows of 4096 -> 4096 39.3 us,
// by tiles 46.0, each workgroup's rows split in it 65.5; 1976 by tiles 148).
constexpr int kMidCopies = 6;
constexpr int kMidUnitBytes = kMidCopies * 1024;

struct MidArgs {
    TileArgs t;
    int32_t splits, tiles;  // S, P
};

template <bool LEAST, bool GATED, int MT>
__global__ __launch_bounds__(kFewThreads, 2) void q4_mid_kernel(MidArgs f) {
    const TileArgs &t = f.t;
    const Q4Args &a = t.a;
    constexpr int kSize = LEAST ? 20 : 18;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, h = lane >> 5;
    const int S = f.splits, P = f.tiles;
    const int split = wave & (S - 1), tile = wave / S;
    const int blocks = t.blocks;
    const int units = (blocks + kUnit - 1) / kUnit;
    const int outs = GATED ? P / 2 : P;  // tiles of the output
    const int columns = static_cast<int>(GATED ? a.half : a.N);
    const int n0 = static_cast<int>(blockIdx.x) * (32 * outs);
    const auto weights = [&](int c) {  // row c of the wave's tile, or the last there is
        const bool second = GATED && tile >= outs;
        const int n = n0 + 32 * (second ? tile - outs : tile) + c;
        return a.w + ((n < columns ? n : columns - 1) + (second ? columns : 0)) * a.row_bytes;
    };
    const uint8_t *source[kMidCopies];
    int skip[kMidCopies], piece[kMidCopies];
#pragma unroll
    for (int c = 0; c < kMidCopies; ++c) {
        const int slot = 64 * c + lane, row = slot / kPieces < 32 ? slot / kPieces : 31;
        const uint8_t *at = weights(row);
        skip[c] = static_cast<int>(reinterpret_cast<uintptr_t>(at) & 15);
        source[c] = at - skip[c];
        piece[c] = 16 * (slot - kPieces * row);
    }
    char *ring = lds + wave * (2 * kMidUnitBytes);
    const auto copy_unit = [&](int u, int buffer) {
        const int count = blocks - kUnit * u < kUnit ? blocks - kUnit * u : kUnit;
#pragma unroll
        for (int c = 0; c < kMidCopies; ++c) {
            const int last = (skip[c] + kSize * count - 1) & ~15;
            fetch16(source[c] + u * (kUnit * kSize) + (piece[c] < last ? piece[c] : last),
                    lds_address(ring) + buffer * kMidUnitBytes + 1024 * c);
        }
    };
    if (split < units) copy_unit(split, 0);
    if (split + S < units) copy_unit(split + S, 1);
    // Words h and 2 + h of this lane's row, of the first block and the second.
    const char *mine = ring + 16 * kPieces * col + static_cast<int>(reinterpret_cast<uintptr_t>(weights(col)) & 15);
    const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(mine + kSize - 16) & 2);
    const char *words[2] = {mine + kSize - 16 + 4 * h - odd, mine + 2 * kSize - 16 + 4 * h - (LEAST ? odd : 2 - odd)};
    const uint32_t shift[2] = {8u * odd, LEAST ? 8u * odd : 16u - 8u * odd};
    const uint32_t magic = opaque(kMagic);
    const char *numbers = t.numbers + static_cast<int64_t>(blockIdx.y) * MT * kNumbersBytes + 16 * lane;
    const int64_t numbers_step = t.row_tiles * kNumbersBytes;
    struct Numbers {
        half8 n[MT][2][2];  // [32 rows][half of the block][hi, lo]
    };
    const auto load_numbers = [&](int b, Numbers &o) {
        const char *from = numbers + (b < blocks ? b : blocks - 1) * numbers_step;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int p = 0; p < 4; ++p) o.n[i][p >> 1][p & 1] = *reinterpret_cast<const half8 *>(from + 4096 * i + 1024 * p);
    };
    float16v acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = float16v{};
    // x of the next kAheadX blocks: those past a unit's are the wave's next
    // unit's, asked for before that one's successor is copied, behind which
    // they would wait.
    constexpr int kAheadX = 4;
    Numbers x[kAheadX];
#pragma unroll
    for (int i = 0; i < kAheadX; ++i) load_numbers(kUnit * split + i, x[i]);
    int buffer = 0;
#pragma unroll 1
    for (int u = split; u < units; u += S) {
        if (u + S < units) {
            fetched<kMidCopies>();
        } else {
            fetched<0>();
        }
        const int count = blocks - kUnit * u < kUnit ? blocks - kUnit * u : kUnit;
        const char *row = mine + buffer * kMidUnitBytes;
        const auto add_block = [&](int i, const Numbers &x) {
            const uint32_t *at = reinterpret_cast<const uint32_t *>(words[i & 1] + buffer * kMidUnitBytes + kSize * (i & ~1));
            _Float16 d;
            __builtin_memcpy(&d, row + kSize * i, 2);
            half8 v[2];
#pragma unroll
            for (int s = 0; s < 2; ++s)
                v[s] = widen(__builtin_amdgcn_alignbit(at[2 * s + 1], at[2 * s], shift[i & 1]), magic);
            const float scale = static_cast<float>(d);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                float16v p = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.n[m][0][1], v[0], float16v{}, 0, 0, 0);
                p = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.n[m][1][1], v[1], p, 0, 0, 0);
                p = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.n[m][0][0], v[0], p, 0, 0, 0);
                p = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.n[m][1][0], v[1], p, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[m][e] = __builtin_fmaf(scale, p[e], acc[m][e]);
            }
        };
#pragma unroll
        for (int i = 0; i < kUnit; ++i) {
            if (i < count) add_block(i, x[i % kAheadX]);
            load_numbers(i < kAheadX ? kUnit * u + i + kAheadX : kUnit * (u + S) + i - kAheadX, x[i % kAheadX]);
        }
        if constexpr (LEAST) {
            // Lane 32 h + row: the offsets of blocks 4 h .. 4 h + 3.
            typedef short short4v __attribute__((ext_vector_type(4)));
            short4v q[3];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = 4 * h + j;
                float c = 0.0f;
                if (k < count) {
                    _Float16 d, least;
                    __builtin_memcpy(&d, row + kSize * k, 2);
                    __builtin_memcpy(&least, row + kSize * k + 2, 2);
                    c = __builtin_fmaf(8.0f, static_cast<float>(d), static_cast<float>(least));
                }
                __bf16 parts[3];
                split_bf16(c, parts);
#pragma unroll
                for (int p = 0; p < 3; ++p) q[p][j] = __builtin_bit_cast(short, parts[p]);
            }
            const char *sums = t.sums + ((u >> 2) * static_cast<int64_t>(t.row_tiles) + blockIdx.y * MT) * kOffsetsBytes +
                               ((u >> 1) & 1) * 3072 + ((u & 1) * 32 + col) * 16 + 8 * h;
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                short4v s[3];
#pragma unroll
                for (int p = 0; p < 3; ++p) s[p] = *reinterpret_cast<const short4v *>(sums + m * kOffsetsBytes + 1024 * p);
#pragma unroll
                for (int total = 2; total >= 0; --total)
#pragma unroll
                    for (int p = 0; p <= total; ++p)
                        acc[m] = __builtin_amdgcn_mfma_f32_32x32x8bf16_1k(s[p], q[total - p], acc[m], 0, 0, 0);
            }
        }
        if (u + 2 * S < units) {
            // The unit is read: the one two on takes its place.
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
            copy_unit(u + 2 * S, buffer);
        }
        buffer ^= 1;
    }
    lds_barrier();
    float *sums = reinterpret_cast<float *>(lds);  // [split][tile][32 rows][register][lane]
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 16; ++e) sums[(((split * P + tile) * MT + m) * 16 + e) * 64 + lane] = acc[m][e];
    lds_barrier();
    constexpr int kTile = MT * 1024;
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * (32 * MT);
    const auto place = [&](int at, int64_t &m, int &out) {
        m = m0 + 32 * ((at >> 10) % MT) + tile_row((at >> 6) & 15) + 4 * ((at >> 5) & 1);
        out = n0 + 32 * (at / kTile) + (at & 31);
        return t.back[m < a.M ? m : a.M - 1];
    };
    if (outs == 1) {
        write_outputs<GATED, kTile / kFewThreads>(a, sums, S, P * kTile, kTile, tid, columns, place, kFewThreads);
    } else {
        write_outputs<GATED, 8>(a, sums, S, P * kTile, outs * kTile, tid, columns, place, kFewThreads);
    }
}

// Splits of K until every wave of the device has one.
int mid_splits(int64_t M, int64_t N, int64_t K, bool gated) {
    const int64_t waves = static_cast<int64_t>(compute_units()) * kFewWaves, units = ceil_div(K / kBlock, kUnit);
    const int64_t tiles = ceil_div(N, 32) * ceil_div(M, M <= 32 ? 32 : 64);
    int splits = 1;
    while (splits < (gated ? 4 : 8) && tiles * splits * 2 <= waves && splits < units) splits *= 2;
    return splits;
}

template <bool LEAST, bool GATED, int MT>
hipError_t launch_mid(const TileArgs &t, hipStream_t stream) {
    constexpr int kLds = kFewWaves * 2 * kMidUnitBytes;
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&q4_mid_kernel<LEAST, GATED, MT>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
    if (attr != hipSuccess) return attr;
    const int64_t columns = GATED ? t.a.half : t.a.N, rows = ceil_div(t.a.M, 32 * MT);
    const int splits = mid_splits(t.a.M, t.a.N, t.a.K, GATED);
    const MidArgs f{t, splits, kFewWaves / splits};
    const dim3 grid(static_cast<uint32_t>(ceil_div(columns, 32 * (GATED ? f.tiles / 2 : f.tiles))), static_cast<uint32_t>(rows));
    SDHIP_LAUNCH((q4_mid_kernel<LEAST, GATED, MT>), grid, dim3(kFewThreads), kLds, stream, f);
    return hipGetLastError();
}

// The work buffer's parts.
struct TilesWork {
    size_t numbers, words, back, sums, offsets, bytes;
    int64_t row_tiles, column_tiles, blocks, groups;
};

// With `weights` those too are laid out, for the tiles.
TilesWork tiles_work(int64_t M, int64_t N, int64_t half, int64_t K, bool least, bool weights) {
    TilesWork w{};
    // Whole workgroups' tiles, whichever shape is taken: 64 or 128 rows by 128
    // or 192.
    w.row_tiles = round_up(ceil_div(M, kRowsTile), 4);
    w.column_tiles = !weights ? 0 : round_up(half ? 2 * ceil_div(half, kRowsTile) : ceil_div(N, kRowsTile), 12);
    w.blocks = K / kBlock;
    w.groups = least ? ceil_div(w.blocks, 32) : 0;
    size_t at = 0;
    const auto take = [&](int64_t bytes) {
        const size_t from = at;
        at += static_cast<size_t>(round_up(bytes, 256));
        return from;
    };
    w.numbers = take(w.blocks * w.row_tiles * kNumbersBytes);
    w.words = take(w.blocks * w.column_tiles * kWordsBytes + 1024);  // the last run's copies end past it
    w.back = take(w.row_tiles * kRowsTile * 4);
    w.sums = take(w.groups * w.row_tiles * kOffsetsBytes);
    w.offsets = take(w.groups * w.column_tiles * kOffsetsBytes);
    w.bytes = at;
    return w;
}

// Which kernels a product of these extents takes, gated or not, numbered as
// the q4_form tuning asks for them.
enum class Form { few = 1, between, tiles4, tiles8, tiles64, tiles192 };

// The operands laid out in the work buffer.
template <bool LEAST, bool GATED>
hipError_t lay_out(const Q4Args &a, void *work, bool weights, TileArgs &t, hipStream_t stream) {
    const TilesWork w = tiles_work(a.M, a.N, a.half, a.K, LEAST, weights);
    t = TileArgs{};
    t.a = a;
    char *p = static_cast<char *>(work);
    t.numbers = p + w.numbers;
    t.words = p + w.words;
    t.back = reinterpret_cast<float *>(p + w.back);
    t.sums = p + w.sums;
    t.offsets = p + w.offsets;
    t.blocks = static_cast<int32_t>(w.blocks);
    t.groups = static_cast<int32_t>(w.groups);
    t.row_tiles = static_cast<int32_t>(w.row_tiles);
    t.column_tiles = static_cast<int32_t>(w.column_tiles);
    t.x_groups = static_cast<int32_t>(ceil_div(a.M, kOperandRows));
    const int64_t tiles = !weights ? 0 : GATED ? 2 * ceil_div(a.half, kRowsTile) : ceil_div(a.N, kRowsTile);
    const int64_t pairs = ceil_div(w.blocks, 32);
    SDHIP_LAUNCH((q4_operands_kernel<LEAST, GATED>), dim3(static_cast<uint32_t>(t.x_groups + tiles * pairs)),
                 dim3(kOperandThreads), 0, stream, t);
    return hipGetLastError();
}

template <bool LEAST, bool GATED>
hipError_t between_rows(const Q4Args &a, void *work, hipStream_t stream) {
    TileArgs t;
    if (const hipError_t e = lay_out<LEAST, GATED>(a, work, false, t, stream); e != hipSuccess) return e;
    return a.M <= 32 ? launch_mid<LEAST, GATED, 1>(t, stream) : launch_mid<LEAST, GATED, 2>(t, stream);
}

template <bool LEAST, bool GATED>
hipError_t many_rows(const Q4Args &a, Form form, void *work, hipStream_t stream) {
    TileArgs t;
    if (const hipError_t e = lay_out<LEAST, GATED>(a, work, true, t, stream); e != hipSuccess) return e;
    switch (form) {
    case Form::tiles4:
        return launch_tiles<LEAST, GATED, 2, 2, 1, 2>(t, stream);
    case Form::tiles8:
        return launch_tiles<LEAST, GATED, 2, 2, 2, 2>(t, stream);
    case Form::tiles192:
        if constexpr (!GATED) return launch_tiles<LEAST, GATED, 1, 2, 4, 3>(t, stream);
        [[fallthrough]];
    default:
        return launch_tiles<LEAST, GATED, 1, 2, 4, 2>(t, stream);
    }
}

// Up to 16 rows need no work buffer; more go by the form of the least time, in
// us: within 6 to 14 % of what 300 calls of 17 .. 8192 rows took, 320 -> 320 to 4096
// -> 16384, and the choices by it 1 % slower than the fastest of all.  Tiles of
// 192 are not paired for the gated product.
Form form_of(int64_t M, int64_t N, int64_t K, bool gated) {
    const int asked = tuning().q4_form;
    // A launch holds 65535 groups of rows at most.
    if (asked > 0 && !(asked == 1 && M > 16 * 65535) && !(asked == 2 && M > 32 * 65535) && !(asked == 6 && gated)) {
        return static_cast<Form>(asked);
    }
    if (M <= 16) return Form::few;
    const float cus = static_cast<float>(compute_units()), blocks = static_cast<float>(K / kBlock);
    const float x = static_cast<float>(M) * static_cast<float>(K) * 1e-6f, w = static_cast<float>(N) * static_cast<float>(K) * 1e-6f;
    Form best = Form::few;
    float least = 0.0f;
    const auto take = [&](Form form, float time) {
        if (least == 0.0f || time < least) {
            best = form;
            least = time;
        }
    };
    // A CU's workgroups, one after another, of `count`.
    const auto rounds = [&](int64_t count) { return std::ceil(static_cast<float>(count) / cus); };
    if (M <= 16 * 65535) take(Form::few, few_shape(M, N, K, gated).time);
    if (M <= 32 * 65535) {
        // x is laid out; then by units of a wave's, of 32 rows of x or 64.
        const int64_t splits = mid_splits(M, N, K, gated);
        const float units = static_cast<float>(ceil_div(ceil_div(K / kBlock, kUnit), splits));
        const int64_t groups = ceil_div(M, M <= 32 ? 32 : 64) * ceil_div(ceil_div(N, 32) * splits, kFewWaves);
        take(Form::between, 2.0f * x + rounds(groups) * (M <= 32 ? 6.5f + 5.0f * units : 9.0f + 7.0f * units));
    }
    // Both are laid out.  Tiles of 128 x 128 by four waves are two a CU, each all
    // of K, and the two do not wait at one barrier (1976 rows of 1280 -> 2 x 5120
    // gated 126 us, by eight waves 142); by eight waves, or of 64 rows, they are
    // split along K inside a workgroup (1976 rows of 5120 -> 1280, tiles that
    // leave some CUs without one: 128 x 128 by four waves 99.6 us, by eight 87.8, 64
    // x 128 99.1, 64 x 192 78.4; 988 rows of 1280 -> 1280 35.4, 31.2, 23.9, 29.1).
    const float both = 1.9f * x + 0.3f * w;
    const float of128 = rounds(ceil_div(M, 128) * ceil_div(N, 128)), of64 = rounds(ceil_div(M, 64) * ceil_div(N, 128));
    const float of192 = rounds(ceil_div(M, 64) * ceil_div(N, 192));
    take(Form::tiles4, 4.2f + both + 8.5f * std::ceil(of128 / 2.0f) + 0.46f * blocks * of128);
    take(Form::tiles8, 3.0f + both + of128 * (8.7f + 0.8f * std::ceil(blocks / 2.0f)));
    take(Form::tiles64, 4.5f + both + of64 * (6.0f + 0.92f * std::ceil(blocks / 4.0f)));
    if (!gated) take(Form::tiles192, 4.7f + both + of192 * (10.2f + 1.12f * std::ceil(blocks / 4.0f)));
    return best;
}

}  // namespace

size_t q4_work_size(int64_t M, int64_t N, int64_t K, bool least) {
    const auto bytes = [&](bool gated) -> size_t {
        const Form form = form_of(M, N, K, gated);
        return form == Form::few ? 0 : tiles_work(M, N, gated ? N / 2 : 0, K, least, form != Form::between).bytes;
    };
    // The plain and the gated product of one size take one size of buffer.
    const size_t plain = bytes(false), gated = N % 2 == 0 ? bytes(true) : 0;
    return plain > gated ? plain : gated;
}

template <bool LEAST, bool GATED>
static hipError_t launch_form(const Q4Args &a, void *work, hipStream_t stream) {
    const Form form = form_of(a.M, a.N, a.K, GATED);
    if (form == Form::few) return few_rows<LEAST, GATED>(a, stream);
    if (form == Form::between) return between_rows<LEAST, GATED>(a, work, stream);
    return many_rows<LEAST, GATED>(a, form, work, stream);
}

hipError_t launch_q4_mul_mat(const Q4Args &a, void *work, hipStream_t stream) {
    KernelScope scope(a.half ? "q4.gated" : "q4", stream);
    if (a.half) return a.least ? launch_form<true, true>(a, work, stream) : launch_form<false, true>(a, work, stream);
    return a.least ? launch_form<true, false>(a, work, stream) : launch_form<false, false>(a, work, stream);
}

}  // namespace sdhip
