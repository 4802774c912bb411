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
// most.  The output is (x - mean) / sqrt(variance + eps) in double, rounded once,
// and then the chain.
//
// Bound by memory: x is read twice, the second time from the Infinity Cache where it
// fits, and y written once.

#include "host.h"
#include "norm_last.h"
#include "profile.h"
#include "row_norm.h"

namespace sdhip {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// What a workgroup takes: channels [c0, c1) and pixels [p0, p1) of an image.
struct View {
    int64_t image, p0, p1;
    int c0, c1, g0, groups, chunk;
};

__device__ __forceinline__ View view_of(const GroupNormLastArgs &a) {
    View v;
    const uint32_t item = blockIdx.x / static_cast<uint32_t>(a.chunks);
    v.chunk = static_cast<int>(blockIdx.x - item * static_cast<uint32_t>(a.chunks));
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

struct Sums {
    double first, squares;
};

// The threads' places in a slab: its channels V at a time, kThreads of them a
// pass, by columns of threads, and the pixels by rows of them.
struct Place {
    int columns, rows, row, c, count;  // count: channels of the pass
};

template <int V>
__device__ __forceinline__ Place place_of(const View &v, int from) {
    Place p;
    p.count = v.c1 - from < kThreads * V ? v.c1 - from : kThreads * V;
    p.columns = (p.count + V - 1) / V;
    p.rows = kThreads / p.columns;
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

constexpr int kAhead = 4;  // pixels of a thread that are loaded together

template <int V>
__global__ __launch_bounds__(kThreads) void group_sums_kernel(GroupNormLastArgs a) {
    __shared__ Sums sums[kThreads * V];
    extern __shared__ Sums totals[];  // the slab's groups'
    const View v = view_of(a);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float *x = a.x + v.image * a.ximage;
    const uint32_t per_group = static_cast<uint32_t>(a.per_group);
    for (int g = tid; g < v.groups; g += kThreads) totals[g] = Sums{0.0, 0.0};
    for (int from = v.c0; from < v.c1; from += kThreads * V) {
        const Place at = place_of<V>(v, from);
        const bool in = at.row < at.rows;
        double first[V], squares[V], shift[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            first[i] = squares[i] = shift[i] = 0.0;
            if (in) shift[i] = static_cast<double>(x[static_cast<uint32_t>(at.c + i) / per_group * per_group]);
        }
        const auto add = [&](const float (&q)[V]) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const double d = static_cast<double>(q[i]) - shift[i];
                first[i] += d;
                squares[i] = __builtin_fma(d, d, squares[i]);
            }
        };
        int64_t p = in ? v.p0 + at.row : v.p1;
        const float *from_x = x + at.c;
        for (; p + (kAhead - 1) * at.rows < v.p1; p += kAhead * at.rows) {
            float q[kAhead][V];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) load_channels<V>(from_x + (p + u * at.rows) * a.xpixel, q[u]);
#pragma unroll
            for (int u = 0; u < kAhead; ++u) add(q[u]);
        }
        for (; p < v.p1; p += at.rows) {
            float q[V];
            load_channels<V>(from_x + p * a.xpixel, q);
            add(q);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) sums[tid * V + i] = Sums{first[i], squares[i]};
        __syncthreads();
        // A group's channels of this pass, over all rows, by a wave.
        for (int g = wave; g < v.groups; g += kWaves) {
            const int64_t whole0 = static_cast<int64_t>(v.g0 + g) * a.per_group, whole1 = whole0 + a.per_group;
            const int low = static_cast<int>(whole0 > from ? whole0 - from : 0);
            const int high = static_cast<int>(whole1 < from + at.count ? whole1 - from : at.count);
            if (low >= high) continue;
            double s = 0.0, t = 0.0;
            for (int r = 0; r < at.rows; ++r)
                for (int i = low + lane; i < high; i += 64) {
                    s += sums[r * at.columns * V + i].first;
                    t += sums[r * at.columns * V + i].squares;
                }
            s = wave_sum(s);
            t = wave_sum(t);
            if (lane == 0) {
                totals[g].first += s;
                totals[g].squares += t;
            }
        }
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

struct Stats {
    double mean, scale;
};

__device__ __forceinline__ Stats stats_of(double shift, double first, double squares, double n, float eps) {
    const double variance = (squares - first * (first / n)) / n;
    // Below 0 by rounding alone; a NaN stays one.
    return Stats{shift + first / n, 1.0 / sqrt((variance < 0.0 ? 0.0 : variance) + static_cast<double>(eps))};
}

template <int V>
__global__ __launch_bounds__(kThreads) void group_last_apply_kernel(GroupNormLastArgs a) {
    extern __shared__ Stats stats[];  // the slab's groups'
    const View v = view_of(a);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float *x = a.x + v.image * a.ximage;
    float *y = a.y + v.image * a.yimage;
    for (int g = wave; g < v.groups; g += kWaves) {
        const int64_t group = v.image * a.groups + v.g0 + g;
        const double *from = a.partials + group * a.parts * 2;
        double s = 0.0, t = 0.0;
        for (int i = lane; i < a.parts; i += 64) {
            s += from[2 * i];
            t += from[2 * i + 1];
        }
        s = wave_sum(s);
        t = wave_sum(t);
        const int64_t c = static_cast<int64_t>(v.g0 + g) * a.per_group;
        const int64_t width = c + a.per_group < a.channels ? a.per_group : a.channels - c;
        if (lane == 0) stats[g] = stats_of(a.firsts[group], s, t, static_cast<double>(width) * static_cast<double>(a.pixels), a.eps);
    }
    __syncthreads();
    const uint32_t per_group = static_cast<uint32_t>(a.per_group), width = static_cast<uint32_t>(a.width);
    for (int from = v.c0; from < v.c1; from += kThreads * V) {
        const Place at = place_of<V>(v, from);
        if (at.row >= at.rows) continue;
        Stats mine[V];
#pragma unroll
        for (int i = 0; i < V; ++i) mine[i] = stats[static_cast<uint32_t>(at.c + i) / per_group - v.g0];
        const float *from_x = x + at.c;
        float *to = y + at.c;
        for (int64_t p0 = v.p0 + at.row; p0 < v.p1; p0 += kAhead * at.rows) {
            float q[kAhead][V];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int64_t p = p0 + u * at.rows;
                load_channels<V>(from_x + (p < v.p1 ? p : p0) * a.xpixel, q[u]);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int64_t p = p0 + u * at.rows;
                if (p >= v.p1) continue;
                float r[V];
#pragma unroll
                for (int i = 0; i < V; ++i) r[i] = static_cast<float>((static_cast<double>(q[u][i]) - mine[i].mean) * mine[i].scale);
                const uint32_t i2 = static_cast<uint32_t>(p) / width, i1 = static_cast<uint32_t>(p) - i2 * width;
                apply_chain_block(a.chain, r, [&](int s, int i) {
                    const DevStep &st = a.chain.steps[s];
                    return (at.c + i) * st.nb[0] + i1 * st.nb[1] + i2 * st.nb[2] + v.image * st.nb[3];
                });
                if constexpr (V == 4) {
                    *reinterpret_cast<float4v *>(to + p * a.ypixel) = float4v{r[0], r[1], r[2], r[3]};
                } else {
                    to[p * a.ypixel] = r[0];
                }
            }
        }
    }
}

// Slabs of whole groups, of 64 channels or more and a multiple of 4 of them where
// the channels are; chunks until each CU has four workgroups, of 8 pixels a
// thread at least.
struct Split {
    int64_t slab_groups, slabs, chunks;
};

Split split_of(const GroupNormLastShape &s) {
    Split p;
    int64_t groups = ceil_div(64, s.per_group);
    while (s.channels % 4 == 0 && groups * s.per_group % 4 != 0) ++groups;
    p.slab_groups = groups < s.groups ? groups : s.groups;
    p.slabs = ceil_div(s.groups, p.slab_groups);
    const int64_t rows = kThreads / (p.slab_groups * s.per_group / 4 < kThreads ? p.slab_groups * s.per_group / 4 + 1 : kThreads);
    const int64_t wanted = ceil_div(4 * static_cast<int64_t>(compute_units()), s.images * p.slabs);
    const int64_t most = ceil_div(s.pixels, 8 * rows);
    p.chunks = wanted < most ? wanted : most;
    return p;
}

}  // namespace

size_t group_norm_last_work_size(const GroupNormLastShape &s) {
    return static_cast<size_t>(s.images * s.groups * (2 * split_of(s).chunks + 1)) * sizeof(double);
}

hipError_t launch_group_norm_last(GroupNormLastArgs a, void *work, hipStream_t stream) {
    KernelScope scope("group_norm_last", stream);
    const Split split = split_of({a.channels, a.pixels, a.images, a.groups, a.per_group});
    a.slab_groups = static_cast<int32_t>(split.slab_groups);
    a.slabs = static_cast<int32_t>(split.slabs);
    a.chunks = a.parts = static_cast<int32_t>(split.chunks);
    a.chunk = ceil_div(a.pixels, split.chunks);
    a.partials = static_cast<double *>(work);
    a.firsts = a.partials + 2 * a.images * a.groups * a.chunks;
    const auto quads = [](const void *p, int64_t pixel, int64_t image) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && pixel % 4 == 0 && image % 4 == 0;
    };
    const bool four = a.channels % 4 == 0 && quads(a.x, a.xpixel, a.ximage) && quads(a.y, a.ypixel, a.yimage);
    const size_t sums = split.slab_groups * sizeof(Sums), stats = split.slab_groups * sizeof(Stats);
    // A launch holds 2^32 - 1 threads at most: 2^23 workgroups of an image or more
    // (one has 2^18 slabs or, where it has several chunks, a few thousand of both).
    const int64_t of_image = split.slabs * split.chunks, most = (int64_t{1} << 23) / of_image;
    for (a.image0 = 0; a.image0 < a.images; a.image0 += most) {
        const int64_t images = a.images - a.image0 < most ? a.images - a.image0 : most;
        const dim3 grid(static_cast<uint32_t>(images * of_image)), block(kThreads);
        if (four) {
            SDHIP_LAUNCH(group_sums_kernel<4>, grid, block, sums, stream, a);
        } else {
            SDHIP_LAUNCH(group_sums_kernel<1>, grid, block, sums, stream, a);
        }
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        if (four) {
            SDHIP_LAUNCH(group_last_apply_kernel<4>, grid, block, stats, stream, a);
        } else {
            SDHIP_LAUNCH(group_last_apply_kernel<1>, grid, block, stats, stream, a);
        }
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace sdhip
