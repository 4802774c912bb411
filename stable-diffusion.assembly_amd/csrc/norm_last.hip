// GROUP_NORM of channels-last tensors with its chain.  A group's numbers are
// `per_group` channels of each pixel of an image, so that a workgroup that reads
// whole lines of memory reads numbers of several groups: it takes a slab of whole
// groups' channels and a chunk of an image's pixels.
//
// Statistics in one pass over x: with c the group's first number, the sums of x - c
// and of (x - c)^2 in double, of which
//     mean = c + S1 / n,  variance = (S2 - S1^2 / n) / n.
// (mean - c)^2 is at most n times the variance, c being one of the group's numbers,
// so that what cancels in the difference costs the variance n 2^-53 of itself at
// most.  The output is (x - mean) / sqrt(variance + eps), the mean in two parts as
// sdhip_norm_residual's (row_norm.h), and then the chain.
//
// Bound by memory.  A slab whose pixels' numbers fit a workgroup's registers takes
// one launch and one read of x; others a launch for the sums and one for the
// outputs, which reads x again, the last chunks first: those the Infinity Cache
// still holds.  1024 x 1024 pixels of 128 channels take 310 us in the kernels (318 a pass
// in a captured graph, 322 with other tensors each time), 5.2 TB/s of the three times that
// they are read or written; 2 x 8 x 8 of 1280 4.7, a launch and three waits one after
// another: x, its sums through LDS, the writes.

#include "host.h"
#include "norm_last.h"
#include "profile.h"
#include "row_norm.h"

namespace sdhip {

namespace {

// What a workgroup takes: channels [c0, c1) and pixels [p0, p1) of an image.
struct View {
    int64_t image, p0, p1;
    int c0, c1, g0, groups, chunk;
};

__device__ __forceinline__ View view_of(const GroupNormLastArgs &a, uint32_t block) {
    View v;
    const uint32_t item = block / static_cast<uint32_t>(a.chunks);
    v.chunk = static_cast<int>(block - item * static_cast<uint32_t>(a.chunks));
    const uint32_t image = item / static_cast<uint32_t>(a.slabs);
    v.image = a.image0 + image;
    const int slab = static_cast<int>(item - image * static_cast<uint32_t>(a.slabs));
    v.g0 = slab * a.slab_groups;
    v.groups = static_cast<int>(a.groups - v.g0 < a.slab_groups ? a.groups - v.g0 : a.slab_groups);
    v.c0 = v.g0 * static_cast<int>(a.per_group);
    const int64_t c1 = static_cast<int64_t>(v.g0 + v.groups) * a.per_group;
    v.c1 = static_cast<int>(c1 < a.channels ? c1 : a.channels);
    v.p0 = v.chunk * a.chunk;
    v.p1 = v.p0 + a.chunk < a.pixels ? v.p0 + a.chunk : a.pixels;
    return v;
}

// The T threads' places in a slab: its channels V at a time, T of them a pass, by
// columns of threads, and the pixels by rows of them.
struct Place {
    int columns, rows, row, c, count;  // count: channels of the pass
};

template <int V, int T>
__device__ __forceinline__ Place place_of(const View &v, int from) {
    Place p;
    p.count = v.c1 - from < T * V ? v.c1 - from : T * V;
    p.columns = (p.count + V - 1) / V;
    p.rows = T / p.columns;
    p.row = static_cast<int>(threadIdx.x) / p.columns;
    p.c = from + (static_cast<int>(threadIdx.x) - p.row * p.columns) * V;
    return p;
}

template <int V>
__device__ __forceinline__ void load_channels(const float *at, float (&q)[V]) {
    if constexpr (V == 4) {
        const float4v four = *reinterpret_cast<const float4v *>(at);
#pragma unroll
        for (int i = 0; i < V; ++i) q[i] = four[i];
    } else {
        q[0] = at[0];
    }
}

struct Sums {
    double first, squares;
};

// The first channel of channel c's group, and of that of c + i, i < V: a division
// for all of them.
__device__ __forceinline__ int first_of(int c, uint32_t per_group) {
    return static_cast<int>(static_cast<uint32_t>(c) / per_group * per_group);
}
template <int V>
__device__ __forceinline__ int at_of(int first, int c, int i, uint32_t per_group) {
    const int n = static_cast<int>(per_group);
    if (n >= V) return c + i - first < n ? first : first + n;
    while (first + n <= c + i) first += n;
    return first;
}

// The sums of V channels of a thread, of x less the channel's group's first number: U
// channels of one group together where the groups are of multiples of U (which leaves a
// U-th of them to add up through LDS: 2 x 16 x 16 x 1280 10.4 us, so 8.3).
template <int V, int U>
struct Channels {
    static constexpr int kUnits = V / U;
    double first[kUnits], squares[kUnits], shift[kUnits];
    __device__ __forceinline__ void begin(const float *x, int c, uint32_t per_group, bool in) {
        const int of = first_of(c, per_group);
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            first[i] = squares[i] = shift[i] = 0.0;
            if (in) shift[i] = static_cast<double>(x[at_of<V>(of, c, i * U, per_group)]);
        }
    }
    __device__ __forceinline__ void add(const float (&q)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const double d = static_cast<double>(q[i]) - shift[i / U];
            first[i / U] += d;
            squares[i / U] = __builtin_fma(d, d, squares[i / U]);
        }
    }
};

// The sum of 8 neighbouring lanes, on all of them.
__device__ __forceinline__ double eight_sum(double v) {
    v += moved<0xb1>(v);          // lanes i ^ 1
    v += moved<0x4e>(v);          // i ^ 2
    return v + moved<0x141>(v);  // 8 lanes mirrored
}

// Adds the threads' sums of a pass's channels, from `from` on, to the slab's
// groups': over the rows by a thread a unit, over a group's units by 8.
template <int V, int U, int T>
__device__ __forceinline__ void add_up(const Channels<V, U> &mine, const View &v, const Place &at, int from, uint32_t per_group,
                                       Sums *sums, Sums *totals) {
    constexpr int kUnits = V / U;
    const int tid = threadIdx.x, units = at.count / U;
    __syncthreads();  // the pass before is added up
    if (at.row < at.rows) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) sums[tid * kUnits + i] = Sums{mine.first[i], mine.squares[i]};
    }
    __syncthreads();
    // The rows of a unit in two rounds: each `step`-th by a thread of their own where
    // there are threads for that, then `step` of them.
    const int pitch = at.columns * kUnits;
    const int most = T / units;
    int step = 1;
    while (step < most && step * step < at.rows) ++step;
    for (int i = tid; i < units * step; i += T) {
        const int r0 = i / units, c = i - r0 * units;
        Sums s = sums[r0 * pitch + c];
#pragma unroll 4
        for (int r = r0 + step; r < at.rows; r += step) {
            const Sums o = sums[r * pitch + c];
            s.first += o.first;
            s.squares += o.squares;
        }
        sums[r0 * pitch + c] = s;
    }
    __syncthreads();
    for (int c = tid; step > 1 && c < units; c += T) {
        Sums s = sums[c];
#pragma unroll 4
        for (int r = 1; r < step; ++r) {
            const Sums o = sums[r * pitch + c];
            s.first += o.first;
            s.squares += o.squares;
        }
        sums[c] = s;
    }
    __syncthreads();
    for (int g = tid / 8; g < v.groups; g += T / 8) {
        const int64_t whole0 = static_cast<int64_t>(v.g0 + g) * per_group, whole1 = whole0 + per_group;
        const int low = static_cast<int>(whole0 > from ? whole0 - from : 0);
        const int high = static_cast<int>(whole1 < from + at.count ? whole1 - from : at.count);
        if (low >= high) continue;  // the 8 lanes of a group together
        double s = 0.0, t = 0.0;
        for (int c = low / U + (tid & 7); c < high / U; c += 8) {
            s += sums[c].first;
            t += sums[c].squares;
        }
        s = eight_sum(s);
        t = eight_sum(t);
        if ((tid & 7) == 0) {
            totals[g].first += s;
            totals[g].squares += t;
        }
    }
}

// Of a group's sums over n numbers.
__device__ __forceinline__ Moments moments_of(double shift, double first, double squares, double n, float eps) {
    const double inverse = 1.0 / n, off = first * inverse, variance = (squares - first * off) * inverse;
    // Below 0 by rounding alone; a NaN stays one.
    return moments(SDHIP_ROW_NORM_LAYER, shift + off, variance < 0.0 ? 0.0 : variance, 1.0, eps);
}

// x / (1 + exp(-x)) by the hardware's power of two and reciprocal (one step of single
// precision off at most, two roundings), the exponent's rounding made up for: within 7
// roundings of itself, down to -87.33; below that, where the sum passes 2^126 and its
// reciprocal the least normal number, within |x| 2^-126.  Where the exponent passes 2^7
// the power is an infinity or 0 and stays so: what is made up for would be NaN, an
// infinity times a rounding below 0 or an infinite exponent's own (the comparison is 0.15
// us of 2 x 64 x 64 x 320's 15.8 in a captured graph).  Fewer than half of the operations
// of silu(), which the outputs of a group norm would wait for: 1.2 us of the same.
__device__ __forceinline__ float fast_silu(float x) {
    const float t = -1.44269504088896341f * x, rest = __builtin_fmaf(-1.44269504088896341f, x, -t);
    const float e = __builtin_amdgcn_exp2f(t), low = __builtin_fmaf(-1.925963033500e-8f, x, rest);
    const float power = __builtin_fabsf(t) < 128.0f ? __builtin_fmaf(e, 0.693147180559945f * low, e) : e;
    return x * __builtin_amdgcn_rcpf(power + 1.0f);
}

// An image's group's numbers.
__device__ __forceinline__ double numbers_of(const GroupNormLastArgs &a, int64_t g) {
    const int64_t c = g * a.per_group, width = c + a.per_group < a.channels ? a.per_group : a.channels - c;
    return static_cast<double>(width) * static_cast<double>(a.pixels);
}

// The outputs of a thread's V channels: their statistics, and the scale and shift of
// a chain that is a multiplication, an addition and SiLU, or some of them in that
// order, by one number a channel (and image): held in registers (`plain`).  Any
// other chain reads its operands for each pixel.  (Six steps of any kind in registers
// are 60 KB of instructions, most of them never run and each launch fetched again: the
// outputs of 2 x 64 x 64 x 320, 9.5 us in a trace, took three times as long by them.)
template <int V>
struct Outputs {
    Moments stats[V];
    float scale[V], shift[V];
    __device__ __forceinline__ void operands(const GroupNormLastArgs &a, const View &v, int c) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            scale[i] = 1.0f;
            shift[i] = 0.0f;
        }
        if (a.plain & kPlainMul) load(a.chain.steps[0], v, c, scale);
        if (a.plain & kPlainAdd) load(a.chain.steps[a.plain & kPlainMul ? 1 : 0], v, c, shift);
    }
    __device__ __forceinline__ void statistics(const GroupNormLastArgs &a, const Moments *of, const View &v, int c) {
        const uint32_t per_group = static_cast<uint32_t>(a.per_group), g = static_cast<uint32_t>(c) / per_group;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            // The group of c + i: c's or, V being less than its channels, the next; else divided.
            const uint32_t mine = per_group < V ? static_cast<uint32_t>(c + i) / per_group : c + i < static_cast<int>((g + 1) * per_group) ? g : g + 1;
            stats[i] = of[mine - v.g0];
        }
    }
    __device__ __forceinline__ void load(const DevStep &st, const View &v, int c, float (&o)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = st.operand[(c + i) * st.nb[0] + v.image * st.nb[3]];
    }
    __device__ __forceinline__ void write(const GroupNormLastArgs &a, const View &v, int c, int64_t p, const float (&q)[V]) const {
        float r[V];
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = normed(q[i], stats[i]);
        if (a.plain) {
            // Times 1 and plus 0 where there is no such step: the same number, but for the
            // sign of a zero.
#pragma unroll
            for (int i = 0; i < V; ++i) r[i] = __fadd_rn(__fmul_rn(r[i], scale[i]), shift[i]);
            if (a.plain & kPlainSilu) {
#pragma unroll
                for (int i = 0; i < V; ++i) r[i] = fast_silu(r[i]);
            }
        } else if (a.chain.count > 0) {
            const uint32_t width = static_cast<uint32_t>(a.width);
            const uint32_t i2 = static_cast<uint32_t>(p) / width, i1 = static_cast<uint32_t>(p) - i2 * width;
            apply_chain_block(a.chain, r, [&](int s, int i) {
                const DevStep &st = a.chain.steps[s];
                return (c + i) * st.nb[0] + i1 * st.nb[1] + i2 * st.nb[2] + v.image * st.nb[3];
            });
        }
        float *to = a.y + v.image * a.yimage + p * a.ypixel + c;
        if constexpr (V == 4) {
            *reinterpret_cast<float4v *>(to) = float4v{r[0], r[1], r[2], r[3]};
        } else {
            to[0] = r[0];
        }
    }
};

constexpr int kThreads = 256;
constexpr int kAhead = 4;  // pixels of a thread that are loaded together

// The sums of a slab's groups over a chunk of pixels.
template <int V, int U>
__global__ __launch_bounds__(kThreads) void group_last_sums_kernel(GroupNormLastArgs a) {
    __shared__ Sums sums[kThreads * (V / U)];
    extern __shared__ Sums totals[];  // the slab's groups'
    const View v = view_of(a, blockIdx.x);
    const int tid = threadIdx.x;
    const float *x = a.x + v.image * a.ximage;
    const uint32_t per_group = static_cast<uint32_t>(a.per_group);
    for (int g = tid; g < v.groups; g += kThreads) totals[g] = Sums{0.0, 0.0};
    for (int from = v.c0; from < v.c1; from += kThreads * V) {
        const Place at = place_of<V, kThreads>(v, from);
        const bool in = at.row < at.rows;
        Channels<V, U> mine;
        mine.begin(x, at.c, per_group, in);
        const float *from_x = x + at.c;
        int64_t p = in ? v.p0 + at.row : v.p1;
        for (; p + (kAhead - 1) * at.rows < v.p1; p += kAhead * at.rows) {
            float q[kAhead][V];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) load_channels<V>(from_x + (p + u * at.rows) * a.xpixel, q[u]);
#pragma unroll
            for (int u = 0; u < kAhead; ++u) mine.add(q[u]);
        }
        for (; p < v.p1; p += at.rows) {
            float q[V];
            load_channels<V>(from_x + p * a.xpixel, q);
            mine.add(q);
        }
        add_up<V, U, kThreads>(mine, v, at, from, per_group, sums, totals);
    }
    __syncthreads();
    for (int g = tid; g < v.groups; g += kThreads) {
        const int64_t group = v.image * a.groups + v.g0 + g;
        double *to = a.partials + (group * a.chunks + v.chunk) * 2;
        to[0] = totals[g].first;
        to[1] = totals[g].squares;
        // For the outputs, which may be written over it.
        if (v.chunk == 0) a.firsts[group] = static_cast<double>(x[static_cast<int64_t>(v.g0 + g) * a.per_group]);
    }
}

constexpr int kMostParts = 256;  // that every workgroup of outputs adds up

// The sum of `L` neighbouring lanes, 32 or 64, on all of them.
template <int L>
__device__ __forceinline__ double lanes_sum(double v) {
    if constexpr (L == 64) return wave_sum(v);
    v = eight_sum(v);
    v += moved<0x140>(v);  // 16 lanes mirrored
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    uint32_t low[2] = {static_cast<uint32_t>(u), static_cast<uint32_t>(u)};
    uint32_t high[2] = {static_cast<uint32_t>(u >> 32), static_cast<uint32_t>(u >> 32)};
    swap16(low[0], low[1]);
    swap16(high[0], high[1]);
    return __builtin_bit_cast(double, static_cast<uint64_t>(high[0]) << 32 | low[0]) +
           __builtin_bit_cast(double, static_cast<uint64_t>(high[1]) << 32 | low[1]);
}

// The statistics of a slab's groups from their parts' sums, L lanes a group, each
// with all of its parts' loads under way together (one after another, a wave a group:
// 2 x 64 x 64 x 320 15.7 us, so 14.2).
template <int L>
__device__ __forceinline__ void join(const GroupNormLastArgs &a, const View &v, Moments *stats) {
    constexpr int kLoads = kMostParts / L;
    const int tid = threadIdx.x, lane = tid % L;
    for (int g = tid / L; g < v.groups; g += kThreads / L) {
        const int64_t group = v.image * a.groups + v.g0 + g;
        const double2 *from = reinterpret_cast<const double2 *>(a.partials) + group * a.parts;
        const double c = a.firsts[group];
        double2 sums[kLoads];
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            sums[u] = double2{0.0, 0.0};
            if (u * L < a.parts) sums[u] = from[lane + u * L < a.parts ? lane + u * L : 0];
        }
        double first = 0.0, squares = 0.0;
#pragma unroll
        for (int u = 0; u < kLoads; ++u) {
            first += lane + u * L < a.parts ? sums[u].x : 0.0;
            squares += lane + u * L < a.parts ? sums[u].y : 0.0;
        }
        first = lanes_sum<L>(first);
        squares = lanes_sum<L>(squares);
        if (lane == 0) stats[g] = moments_of(c, first, squares, numbers_of(a, v.g0 + g), a.eps);
    }
}

// The statistics of all groups, a workgroup each, where their parts are too many for
// every workgroup of outputs to add up.
__global__ __launch_bounds__(256) void group_last_join_kernel(GroupNormLastArgs a) {
    __shared__ Sums sums[4];
    const int64_t image = blockIdx.x / a.groups, g = blockIdx.x - image * a.groups, group = (a.image0 + image) * a.groups + g;
    const double c = a.firsts[group];
    const double2 *from = reinterpret_cast<const double2 *>(a.partials) + group * a.parts;
    Sums mine{0.0, 0.0};
#pragma unroll 4
    for (int i = threadIdx.x; i < a.parts; i += 256) {
        mine.first += from[i].x;
        mine.squares += from[i].y;
    }
    mine = Sums{wave_sum(mine.first), wave_sum(mine.squares)};
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x / 64] = mine;
    __syncthreads();
    if (threadIdx.x != 0) return;
    const Moments s = moments_of(c, (sums[0].first + sums[1].first) + (sums[2].first + sums[3].first),
                             (sums[0].squares + sums[1].squares) + (sums[2].squares + sums[3].squares), numbers_of(a, g), a.eps);
    reinterpret_cast<Moments *>(a.joined)[group] = s;
}

// The outputs of a slab's channels and a chunk of pixels.
template <int V>
__global__ __launch_bounds__(kThreads, 4) void group_last_apply_kernel(GroupNormLastArgs a) {
    extern __shared__ Moments stats[];  // the slab's groups'
    // The last chunks that the sums read, first.
    const View v = view_of(a, gridDim.x - 1 - blockIdx.x);
    const int tid = threadIdx.x;
    const float *x = a.x + v.image * a.ximage;
    Outputs<V> out;
    float q[kAhead][V];
    const auto load = [&](const Place &at, int64_t p0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int64_t p = p0 + u * at.rows;
            load_channels<V>(x + at.c + (p < v.p1 ? p : v.p0) * a.xpixel, q[u]);
        }
    };
    // The first pixels and the operands are under way while the statistics are joined.
    {
        const Place at = place_of<V, kThreads>(v, v.c0);
        if (at.row < at.rows) {
            out.operands(a, v, at.c);
            load(at, v.p0 + at.row);
        }
    }
    if (a.joined != nullptr) {
        for (int g = tid; g < v.groups; g += kThreads) {
            stats[g] = reinterpret_cast<const Moments *>(a.joined)[v.image * a.groups + v.g0 + g];
        }
    } else {
        if (v.groups <= 4) {
            join<64>(a, v, stats);
        } else {
            join<32>(a, v, stats);
        }
    }
    __syncthreads();
    for (int from = v.c0; from < v.c1; from += kThreads * V) {
        const Place at = place_of<V, kThreads>(v, from);
        if (at.row >= at.rows) continue;
        if (from > v.c0) {
            out.operands(a, v, at.c);
            load(at, v.p0 + at.row);
        }
        out.statistics(a, stats, v, at.c);
        for (int64_t p0 = v.p0 + at.row; p0 < v.p1; p0 += kAhead * at.rows) {
            if (p0 > v.p0 + at.row) load(at, p0);
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int64_t p = p0 + u * at.rows;
                if (p < v.p1) out.write(a, v, at.c, p, q[u]);
            }
        }
    }
}

// Sums and outputs in one launch: a workgroup holds a slab's numbers of an image,
// R pixels a thread.
template <int V, int U, int T, int R>
__global__ __launch_bounds__(T) void group_last_whole_kernel(GroupNormLastArgs a) {
    extern __shared__ Sums sums[];
    Sums *totals = sums + T * (V / U);  // the slab's groups', and then their statistics
    const View v = view_of(a, blockIdx.x);
    const int tid = threadIdx.x;
    const float *x = a.x + v.image * a.ximage;
    const uint32_t per_group = static_cast<uint32_t>(a.per_group);
    const Place at = place_of<V, T>(v, v.c0);
    const bool in = at.row < at.rows;
    const int pixels = static_cast<int>(v.p1);
    float q[R][V];
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int p = at.row + u * at.rows;
        load_channels<V>(x + at.c + (in && p < pixels ? p : 0) * a.xpixel, q[u]);
    }
    Channels<V, U> mine;
    mine.begin(x, at.c, per_group, in);
    Outputs<V> out;
    if (in) out.operands(a, v, at.c);
    // A slab's groups are fewer than the threads.
    const float first = tid < v.groups ? x[static_cast<int64_t>(v.g0 + tid) * a.per_group] : 0.0f;
    if (tid < v.groups) totals[tid] = Sums{0.0, 0.0};
#pragma unroll
    for (int u = 0; u < R; ++u)
        if (in && at.row + u * at.rows < pixels) mine.add(q[u]);
    if (v.groups == 1) {
        // Of one group the sums of all threads, by waves (2 x 8 x 8 x 1280 5.9 us by its
        // channels, so 4.6).
        double one = 0.0, two = 0.0;
#pragma unroll
        for (int i = 0; i < V / U; ++i) {
            one += mine.first[i];
            two += mine.squares[i];
        }
        one = wave_sum(one);
        two = wave_sum(two);
        if ((tid & 63) == 0) sums[tid / 64] = Sums{one, two};
        __syncthreads();  // and x is read, which y may be
        one = two = 0.0;
#pragma unroll
        for (int w = 0; w < T / 64; ++w) {
            one += sums[w].first;
            two += sums[w].squares;
        }
        if (!in) return;
        const Moments m = moments_of(mine.shift[0], one, two, numbers_of(a, v.g0), a.eps);
#pragma unroll
        for (int i = 0; i < V; ++i) out.stats[i] = m;
    } else {
        add_up<V, U, T>(mine, v, at, v.c0, per_group, sums, totals);
        __syncthreads();
        Moments *stats = reinterpret_cast<Moments *>(totals);
        if (tid < v.groups) {
            stats[tid] = moments_of(static_cast<double>(first), totals[tid].first, totals[tid].squares, numbers_of(a, v.g0 + tid), a.eps);
        }
        __syncthreads();  // and x is read, which y may be
        if (!in) return;
        out.statistics(a, stats, v, at.c);
    }
#pragma unroll
    for (int u = 0; u < R; ++u) {
        const int p = at.row + u * at.rows;
        if (p < pixels) out.write(a, v, at.c, p, q[u]);
    }
}

// ------------------------------------------------------------------ the split

// The threads of the one launch, and the numbers of each: as few threads as hold a
// slab's (what a wave does once is as much as five pixels).
struct Whole {
    int threads, numbers;
};
constexpr Whole kWhole[] = {{256, 16}, {512, 16}, {1024, 16}, {1024, 32}};

int64_t gcd(int64_t a, int64_t b) { return b == 0 ? a : gcd(b, a % b); }

// Groups of a slab of `channels` or more of them, beginning at a multiple of V.
int64_t slab_of(const GroupNormLastShape &s, int64_t channels, int v) {
    const int64_t unit = v / gcd(v, s.per_group);
    const int64_t groups = round_up(ceil_div(channels, s.per_group), unit);
    return groups < s.groups ? groups : s.groups;
}

// Rows of T threads by V channels over a slab of so many groups.
int64_t rows_of(const GroupNormLastShape &s, int64_t slab, int64_t threads, int v) {
    const int64_t channels = slab * s.per_group < s.channels ? slab * s.per_group : s.channels, columns = ceil_div(channels, v);
    return columns < threads ? threads / columns : 1;
}

struct Split {
    int v;                       // channels a thread
    int whole;                   // which of kWhole one launch is of, or -1: two launches or three
    int64_t slab, slabs;         // of the sums (or of the one launch)
    int64_t parts;
    int64_t apply, apply_slabs;  // of the outputs
    int64_t chunks;
    bool joined;                 // three launches
};

// By V channels a thread, in one launch slabs of `least` channels or more.
Split split_of(const GroupNormLastShape &s, int v, int64_t least) {
    Split p{};
    p.v = v;
    const int64_t cus = compute_units();
    p.slab = slab_of(s, least, v);
    p.slabs = ceil_div(s.groups, p.slab);
    for (p.whole = 0; p.whole < 4; ++p.whole) {
        const Whole &w = kWhole[p.whole];
        if (p.slab * s.per_group <= w.threads * v && s.pixels <= w.numbers / v * rows_of(s, p.slab, w.threads, v)) return p;
    }
    p.whole = -1;
    // Whole lines of up to 1024 channels; chunks until each CU has 16 workgroups, three
    // rounds of them, whose last leaves less to wait for than that of 8 (4 x 108 x 183 x
    // 1376 296 us, so 264, 1024 x 1024 x 128 315 and 308), of 8 pixels a thread at least.  None is empty: as many as chunks of the pixels of
    // one of them are (the outputs' kernel reads its chunk's first pixel).
    p.slab = slab_of(s, ceil_div(s.channels, ceil_div(s.channels, 1024)), v);
    p.slabs = ceil_div(s.groups, p.slab);
    const auto chunks = [&](int64_t slab, int64_t slabs, int64_t least) {
        const int64_t wanted = ceil_div(16 * cus, s.images * slabs), most = ceil_div(s.pixels, least * rows_of(s, slab, kThreads, v));
        return ceil_div(s.pixels, ceil_div(s.pixels, wanted < most ? wanted : most));
    };
    p.parts = chunks(p.slab, p.slabs, 8);
    p.joined = p.parts > kMostParts;
    // Where the outputs' workgroups add up the parts, of few groups each.
    p.apply = p.joined ? p.slab : slab_of(s, 64, v);
    p.apply_slabs = ceil_div(s.groups, p.apply);
    p.chunks = chunks(p.apply, p.apply_slabs, 8);
    return p;
}

// Slabs of 64 bytes or more, by four channels a thread where they lie so.  Where that
// leaves half of the CUs without one, slabs of 32 bytes by one launch, by single
// channels where a group is of no multiple of four: a CU's operations, not memory,
// bound the slabs of many numbers (more than 6000; 33 x 24 of 352 11.2 us by 44 channels,
// 8.7 by 11, 3 x 53 x 7 of 288 10.4 and 7.7; 3 x 5 x 40 of 48, by 4800 numbers, 6.4 and
// 7.3), single channels cost more a number, and of 10000 and more as much as two launches
// (2 x 109 x 17 of 288, by 16700, 16.0 us, so 12.2).
Split choose(const GroupNormLastShape &s, bool quads) {
    const Split wide = split_of(s, quads ? 4 : 1, 16);
    const auto numbers = [&](const Split &p) { return p.slab * s.per_group * s.pixels; };
    if (wide.whole >= 0 && (2 * s.images * wide.slabs >= compute_units() || numbers(wide) <= 6000)) return wide;
    const Split narrow = split_of(s, quads && s.per_group % 4 == 0 ? 4 : 1, 8);
    return narrow.whole >= 0 && narrow.slabs > wide.slabs && numbers(narrow) <= 10000 ? narrow : wide;
}

// The chain's steps as a multiplication, an addition and SiLU of one number a
// channel; 0: it is another, or none.
int32_t plain_of(const DevChain &c) {
    int32_t plain = 0;
    for (int s = 0; s < c.count; ++s) {
        const DevStep &st = c.steps[s];
        const int32_t step = st.kind == kMul ? kPlainMul : st.kind == kAdd ? kPlainAdd : kPlainSilu;
        if (plain >= step || (st.kind != kSilu && (st.nb[1] != 0 || st.nb[2] != 0))) return 0;
        plain |= step;
    }
    return plain;
}

size_t work_of(const GroupNormLastShape &s, const Split &p) {
    return p.whole >= 0 ? 0 : static_cast<size_t>(s.images * s.groups * (2 * p.parts + 1 + (p.joined ? 2 : 0))) * sizeof(double);
}

template <int V, int U, int T, int R, class ByImages>
hipError_t launch_whole(ByImages by_images, const Split &split, const GroupNormLastArgs &a, hipStream_t stream) {
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&group_last_whole_kernel<V, U, T, R>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (attr != hipSuccess) return attr;
    return by_images(split.slab, split.slabs, 1, [&](int64_t, dim3 grid, uint32_t lds) {
        SDHIP_LAUNCH((group_last_whole_kernel<V, U, T, R>), grid, dim3(T), static_cast<uint32_t>(T * (V / U) * sizeof(Sums)) + lds, stream, a);
    });
}

template <int V, int U>
hipError_t launch(GroupNormLastArgs a, const Split &split, void *work, hipStream_t stream) {
    // A launch holds 2^32 - 1 threads at most: 2^21 workgroups of an image or more (one
    // has 2^18 slabs or, where it has several chunks, a few thousand of both).
    const auto by_images = [&](int64_t slab, int64_t slabs, int64_t chunks, auto run) {
        a.slab_groups = static_cast<int32_t>(slab);
        a.slabs = static_cast<int32_t>(slabs);
        a.chunks = static_cast<int32_t>(chunks);
        a.chunk = ceil_div(a.pixels, chunks);
        const int64_t most = (int64_t{1} << 21) / (slabs * chunks);
        for (a.image0 = 0; a.image0 < a.images; a.image0 += most) {
            const int64_t images = a.images - a.image0 < most ? a.images - a.image0 : most;
            run(images, dim3(static_cast<uint32_t>(images * slabs * chunks)), static_cast<uint32_t>(slab * sizeof(Sums)));
            if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        }
        return hipSuccess;
    };
    static_assert(sizeof(Sums) == sizeof(Moments));
    if (split.whole == 0) return launch_whole<V, U, kWhole[0].threads, kWhole[0].numbers / V>(by_images, split, a, stream);
    if (split.whole == 1) return launch_whole<V, U, kWhole[1].threads, kWhole[1].numbers / V>(by_images, split, a, stream);
    if (split.whole == 2) return launch_whole<V, U, kWhole[2].threads, kWhole[2].numbers / V>(by_images, split, a, stream);
    if (split.whole == 3) return launch_whole<V, U, kWhole[3].threads, kWhole[3].numbers / V>(by_images, split, a, stream);
    a.parts = static_cast<int32_t>(split.parts);
    a.partials = static_cast<double *>(work);
    double *at = a.partials + 2 * a.images * a.groups * split.parts;
    if (split.joined) {
        a.joined = at;
        at += 2 * a.images * a.groups;
    }
    a.firsts = at;
    hipError_t e = by_images(split.slab, split.slabs, split.parts, [&](int64_t, dim3 grid, uint32_t lds) {
        SDHIP_LAUNCH((group_last_sums_kernel<V, U>), grid, dim3(kThreads), lds, stream, a);
    });
    if (e == hipSuccess && split.joined) {
        e = by_images(1, a.groups, 1, [&](int64_t images, dim3, uint32_t) {
            SDHIP_LAUNCH(group_last_join_kernel, dim3(static_cast<uint32_t>(images * a.groups)), dim3(256), 0, stream, a);
        });
    }
    if (e != hipSuccess) return e;
    return by_images(split.apply, split.apply_slabs, split.chunks, [&](int64_t, dim3 grid, uint32_t lds) {
        SDHIP_LAUNCH(group_last_apply_kernel<V>, grid, dim3(kThreads), lds, stream, a);
    });
}

}  // namespace

size_t group_norm_last_work_size(const GroupNormLastShape &s) {
    // Of either, as the tensors may lie.
    const size_t four = s.channels % 4 == 0 ? work_of(s, choose(s, true)) : 0, one = work_of(s, choose(s, false));
    return four > one ? four : one;
}

hipError_t launch_group_norm_last(GroupNormLastArgs a, void *work, hipStream_t stream) {
    KernelScope scope("group_norm_last", stream);
    a.plain = plain_of(a.chain);
    const auto quads = [](const void *p, int64_t pixel, int64_t image) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && pixel % 4 == 0 && image % 4 == 0;
    };
    const GroupNormLastShape s{a.channels, a.pixels, a.images, a.groups, a.per_group};
    const Split split = choose(s, a.channels % 4 == 0 && quads(a.x, a.xpixel, a.ximage) && quads(a.y, a.ypixel, a.yimage));
    if (split.v == 1) return launch<1, 1>(a, split, work, stream);
    if (a.per_group % 4 == 0) return launch<4, 4>(a, split, work, stream);
    return a.per_group % 2 == 0 ? launch<4, 2>(a, split, work, stream) : launch<4, 1>(a, split, work, stream);
}

}  // namespace sdhip
