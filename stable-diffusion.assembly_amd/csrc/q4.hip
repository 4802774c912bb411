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
// its row's greatest number to [2^14, 2^15): 22 bits of every number within
// 2^28 of the greatest (lo a normal number), 2^-39 of the greatest off at most
// below.  A block's 32 products fill one v_mfma_f32_16x16x32_f16 (two with
// both parts), whose sums in single precision are then scaled by d and added
// up; so no weight is rounded.

#include "host.h"
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

__device__ __forceinline__ void swap32(uint32_t &a, uint32_t &b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}

__device__ __forceinline__ void swap16(uint32_t &a, uint32_t &b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
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

// ------------------------------------------------------------------ copies

// A copy of 16 bytes a lane (1 KB) or 4 into LDS at `to` and on, lane after
// lane.  The compiler does not see these loads, and so does not wait for them
// where it waits for others or reads LDS: what reads them waits (wait_loads).
// Nothing else here uses m0.
__device__ __forceinline__ void fetch16(const void *from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(to)),
                 "v"(from)
                 : "memory");
}
__device__ __forceinline__ void fetch4(const void *from, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(to)),
                 "v"(from)
                 : "memory");
}

__device__ __forceinline__ uint32_t lds_address(const char *p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char *)p));
}

// wait_loads, and no read of LDS before it.
template <int N>
__device__ __forceinline__ void fetched() {
    wait_loads<N>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// ------------------------------------------------------------------ few rows

// Up to 16 rows of x.  A workgroup takes P tiles of 16 rows of the weights
// (with GATED, P / 2 of each half) by S splits of K, a wave each, P S = 8; a
// split is every S-th unit of 8 blocks, and the splits' sums are added at the
// end in their order.
//
// What bounds it is the weights' bytes, each loaded once: a wave has two units
// of them (16 rows, 144 or 160 bytes each) in flight, copied into LDS of its
// own as the 16-byte pieces of memory that hold them, wherever in those a
// row begins (loads of each block by a lane of its own, at even addresses 18
// bytes apart, moved 16384 rows of 4096 at 2.7 TB/s, aligned pieces at 5.3).
// x is copied into LDS before them and split there, a wave taking 512 numbers
// of a row at a time, each such part with a scale of its own and in its own
// place; where x's rows take more than 64 KB, in chunks of K of as many parts
// as fit.  Short calls spend their time on what runs once -- instructions
// fetched, addresses, a barrier -- so little does.  The 16 rows of an MFMA are 4 on each group of lanes, of
// which a result's 4 registers are the sums: up to 4 rows of x are one a group,
// its hi in the first register and its lo in the second, up to 8 two a group,
// so that one MFMA takes both parts; from 9 on two do.
constexpr int kFewWaves = 8;
constexpr int kFewThreads = 64 * kFewWaves;
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
    const int split = wave & (S - 1), tile = wave / S;
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
        for (int u = wave; u < share; u += kFewWaves) {
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
        for (int u = wave; u < share; u += kFewWaves) {
            // A lane's 8 numbers, 4 group .. and 16 + 4 group .. of a block,
            // make way for their hi and their lo.
            char *place = lds + kPartBytes * u + 128 * (lane >> 2) + 16 * (lane & 3);
            const float4v low = *reinterpret_cast<const float4v *>(place);
            const float4v high = *reinterpret_cast<const float4v *>(place + 64);
            uint32_t v = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t p = __builtin_bit_cast(uint32_t, static_cast<float>(low[k])) & 0x7fffffffu;
                const uint32_t q = __builtin_bit_cast(uint32_t, static_cast<float>(high[k])) & 0x7fffffffu;
                v = v > p ? v : p;
                v = v > q ? v : q;
            }
            const uint32_t e = scale_exponent(wave_greatest(v));
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
#pragma unroll 1
    for (int at = tid; at < outs * R * 64; at += kFewThreads) {
        const int row = R * ((at & 63) >> 4) + (at >> 6) % R;
        const int out = n0 + 16 * (at / (64 * R)) + (at & 15);
        if (row >= rows || out >= columns) continue;
        const int64_t m = m0 + row;
        float *y = a.y + m * a.ldy + out;
        float v[GATED ? 2 : 1];
#pragma unroll
        for (int p = 0; p < (GATED ? 2 : 1); ++p) {
            v[p] = 0.0f;
#pragma unroll 1
            for (int u = 0; u < S; ++u) v[p] += sums[(u * P + p * outs) * R * 64 + at];
        }
        if (a.from_redirect) v[0] = *y + v[0];
        if (a.chain.count > 0) {
            uint32_t i1, i2, i3;
            split_index(static_cast<uint32_t>(m), static_cast<uint32_t>(a.ne1), static_cast<uint32_t>(a.ne2), i1, i2, i3);
            apply_chain_block(a.chain, v, [&](int s, int p) {
                const DevStep &st = a.chain.steps[s];
                return (out + p * static_cast<int64_t>(columns)) * st.nb[0] + i1 * st.nb[1] + i2 * st.nb[2] +
                       i3 * st.nb[3];
            });
        }
        *y = GATED ? v[0] * gelu(v[GATED ? 1 : 0]) : v[0];
    }
}

template <bool LEAST, bool GATED, int ROWS>
hipError_t launch_few(const Q4Args &a, hipStream_t stream) {
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&q4_few_kernel<LEAST, GATED, ROWS>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize,
                                                       kFewParts * kPartBytes + kFewWaves * kRing);
    if (attr != hipSuccess) return attr;
    FewArgs f{};
    f.a = a;
    f.splits = 1;
    const int64_t columns = GATED ? a.half : a.N;
    const int64_t tiles = ceil_div(a.N, 16), units = ceil_div(a.K / kBlock, kUnit);
    const int64_t parts = ceil_div(a.K / kBlock, kPart) * ROWS;
    const int64_t chunk = kFewParts / ROWS * kPart / kUnit;
    // Splits until the device's waves all have one, two workgroups a CU.
    const int64_t waves = static_cast<int64_t>(compute_units()) * 2 * kFewWaves;
    const int most = GATED ? 4 : 8;
    while (f.splits < most && tiles * f.splits * 2 <= waves && f.splits < units && f.splits < chunk) f.splits *= 2;
    f.tiles = kFewWaves / f.splits;
    const dim3 grid(static_cast<uint32_t>(ceil_div(columns, 16 * (GATED ? f.tiles / 2 : f.tiles))),
                    static_cast<uint32_t>(ceil_div(a.M, ROWS)));
    f.ring = static_cast<int32_t>(kPartBytes * (parts < kFewParts ? parts : kFewParts));
    f.aligned = reinterpret_cast<uintptr_t>(a.x) % 16 == 0;
    SDHIP_LAUNCH((q4_few_kernel<LEAST, GATED, ROWS>), grid, dim3(kFewThreads),
                 static_cast<uint32_t>(f.ring + kFewWaves * kRing), stream, f);
    return hipGetLastError();
}

template <bool LEAST, bool GATED>
hipError_t few_rows(const Q4Args &a, hipStream_t stream) {
    if (a.M == 1) return launch_few<LEAST, GATED, 1>(a, stream);
    if (a.M == 2) return launch_few<LEAST, GATED, 2>(a, stream);
    if (a.M <= 4) return launch_few<LEAST, GATED, 4>(a, stream);
    if (a.M <= 8) return launch_few<LEAST, GATED, 8>(a, stream);
    return launch_few<LEAST, GATED, 16>(a, stream);
}

}  // namespace

hipError_t launch_q4_mul_mat(const Q4Args &a, hipStream_t stream) {
    KernelScope scope(a.half ? "q4.gated" : "q4", stream);
    if (a.half) return a.least ? few_rows<true, true>(a, stream) : few_rows<false, true>(a, stream);
    return a.least ? few_rows<true, false>(a, stream) : few_rows<false, false>(a, stream);
}

}  // namespace sdhip
