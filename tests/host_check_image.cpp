// The host code of the products of 8-bit floating-point weights, of the rotary positions
// and of GROUP_NORM of channels-last tensors under AddressSanitizer and
// UndefinedBehaviorSanitizer: predicates, work sizes and the entry points' refusals,
// driven with randomized descriptors near what they take, extents up to the largest
// ones and strides of any sign.  What each call answers is checked by the Python tests;
// here any undefined behaviour stops the run.  No call is launched: the entry points
// are reached with operands that they refuse.
//
//   make -C stable-diffusion.assembly_amd host_check && stable-diffusion.assembly_amd/_build/host_check_image [cases [seed]]

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <string>
#include <vector>

#include "../include/sdhip.h"

// The HIP runtime's own allocations live until the process ends.
extern "C" const char *__asan_default_options() { return "detect_leaks=0"; }

namespace {

std::mt19937_64 rng(12345);

template <typename T>
T one_of(std::initializer_list<T> values) {
    return *(values.begin() + rng() % values.size());
}

int64_t pick(std::initializer_list<int64_t> values) { return one_of<int64_t>(values); }

// Host memory the descriptors point into: never read by the calls here.
std::vector<char> arena(1 << 16);

void *place() {
    return rng() % 16 == 0 ? nullptr : arena.data() + (rng() % 256) * 16 + (rng() % 4 == 0 ? rng() % 16 : 0);
}

int64_t large() {
    return pick({INT32_MAX, int64_t{1} << 24, int64_t{1} << 25, (int64_t{1} << 25) + 1, int64_t{1} << 31, int64_t{1} << 40,
                 INT64_MAX, INT64_MIN});
}

int64_t extent() { return rng() % 24 == 0 ? large() : pick({-1, 0, 1, 1, 1, 2, 3, 4, 7, 16, 17, 33, 64, 65, 128, 200, 300, 1000, 2000}); }

int64_t stride() { return rng() % 8 == 0 ? large() : pick({0, 1, 2, 4, 6, 16, 36, 64, 1280, -4, -16}); }

int64_t times(int64_t a, int64_t b) {
    int64_t r;
    return __builtin_mul_overflow(a, b, &r) ? INT64_MAX : r;
}

sdhip_tensor tensor(int32_t type, int64_t size, int64_t n0, int64_t n1, int64_t n2, int64_t n3) {
    sdhip_tensor t{};
    t.type = rng() % 32 ? type : static_cast<int32_t>(pick({0, 1, 2, 256, -1}));
    const int64_t ne[4] = {n0, n1, n2, n3};
    for (int i = 0; i < 4; ++i) t.ne[i] = rng() % 24 ? ne[i] : extent();
    t.nb[0] = rng() % 32 ? size : stride();
    t.nb[1] = rng() % 6 ? times(t.ne[0], size) : stride();
    for (int i = 2; i < 4; ++i) t.nb[i] = rng() % 16 ? times(t.nb[i - 1], t.ne[i - 1]) : stride();
    t.data = place();
    return t;
}

sdhip_tensor floats(int64_t n0, int64_t n1, int64_t n2, int64_t n3) { return tensor(SDHIP_TYPE_F32, 4, n0, n1, n2, n3); }

void wrong(const char *what) {
    std::printf("%s\n", what);
    std::exit(1);
}

// Tensors far from each other, most of the time.
void apart(std::initializer_list<sdhip_tensor *> all) {
    if (rng() % 4 == 0) return;
    int64_t at = 0;
    for (sdhip_tensor *t : all) t->data = reinterpret_cast<void *>(++at << 45);
}

int64_t up(int64_t v) { return v > 0 && v <= INT64_MAX - 127 ? (v + 127) / 128 : v; }

void products() {
    const int64_t k = extent(), n = rng() % 2 ? extent() : times(2, extent()), m = extent();
    const int64_t m2 = rng() % 3 ? 1 : extent(), m3 = rng() % 3 ? 1 : extent();
    sdhip_tensor w = tensor(SDHIP_TYPE_F8_E4M3, 1, k, n, 1, 1), s = floats(up(k), up(n), 1, 1), x = floats(k, m, m2, m3);
    sdhip_tensor y = floats(n, m, m2, m3), out = floats(n / 2, m, m2, m3);
    apart({&w, &s, &x, &y, &out});
    const int taken = sdhip_mul_mat_f8_supported(&w, &s, &x, &y);
    const size_t need = sdhip_mul_mat_f8_work_size(&w, &s, &x, &y);
    if (sdhip_mul_mat_f8_gated_supported(&w, &s, &x, &y, &out) && !taken) wrong("a gated product of a product that is not taken");
    if (!taken && need != 0) wrong("a size for a product that is not taken");
    // Refused for its operands, else for its missing output.
    y.data = out.data = nullptr;
    if (sdhip_mul_mat_f8(&w, &s, &x, &y, nullptr, nullptr, 0, nullptr) == SDHIP_OK ||
        sdhip_mul_mat_f8_gated(&w, &s, &x, &y, nullptr, &out, nullptr, 0, nullptr) == SDHIP_OK) {
        wrong("a product without an output was taken");
    }
}

void turns() {
    const int64_t d = extent(), tokens = extent(), heads = extent(), batch = extent();
    sdhip_rope_axes axes{};
    axes.count = static_cast<int32_t>(rng() % 16 ? 1 + rng() % SDHIP_MAX_AXES : pick({-1, 0, SDHIP_MAX_AXES + 1, INT32_MAX}));
    axes.order = static_cast<int32_t>(rng() % 16 ? rng() % 2 : pick({-1, 2}));
    axes.shared = static_cast<int32_t>(rng() % 2);
    for (int i = 0; i < SDHIP_MAX_AXES; ++i) {
        axes.dims[i] = static_cast<int32_t>(rng() % 16 ? pick({2, 4, 16, 44}) : pick({-2, 0, 3, INT32_MAX - 1}));
        axes.base[i] = one_of<float>({10000.0f, 1.0f, 1e-30f, rng() % 8 ? 100.0f : NAN, rng() % 8 ? 2.0f : -1.0f});
    }
    const bool half = rng() % 2;
    sdhip_tensor x = floats(d, tokens, heads, batch);
    sdhip_tensor y = tensor(half ? SDHIP_TYPE_F16 : SDHIP_TYPE_F32, half ? 2 : 4, d, tokens, heads, batch);
    sdhip_tensor at = floats(axes.count, rng() % 3 ? tokens : 1, 1, rng() % 3 ? batch : 1);
    sdhip_tensor weight = floats(d, 1, rng() % 2 ? heads : 1, 1), bias = floats(d, 1, 1, 1);
    apart({&x, &y, &at, &weight, &bias});
    sdhip_row_norm norm{};
    norm.kind = static_cast<int32_t>(rng() % 16 ? rng() % 3 : pick({-1, 3}));
    norm.weight = rng() % 2 ? &weight : nullptr;
    norm.bias = rng() % 2 ? &bias : nullptr;
    const auto maybe = [&](auto *p) { return rng() % 12 ? p : nullptr; };
    sdhip_rope_supported(maybe(&x), maybe(&norm), maybe(&at), maybe(&axes), maybe(&y));
    y.data = nullptr;
    if (sdhip_rope(&x, &norm, &at, &axes, &y, nullptr) == SDHIP_OK) wrong("positions without an output were taken");
}

void norms() {
    sdhip_tensor x = floats(extent(), extent(), extent(), extent());
    sdhip_tensor y = floats(x.ne[0], x.ne[1], x.ne[2], x.ne[3]);
    apart({&x, &y});
    const int groups = static_cast<int>(rng() % 12 ? 1 + rng() % 64 : pick({-1, 0, INT32_MAX}));
    const int taken = sdhip_group_norm_last_supported(&x, &y, groups);
    if (sdhip_group_norm_last_work_size(&x, &y, groups) != 0 && !taken) wrong("a size for a norm that is not taken");
    y.data = nullptr;
    if (sdhip_group_norm_last(&x, &y, groups, 1e-6f, nullptr, nullptr, 0, nullptr) == SDHIP_OK) {
        wrong("a norm without an output was taken");
    }
}

}  // namespace

int main(int argc, char **argv) {
    const int cases = argc > 1 ? std::atoi(argv[1]) : 20000;
    if (argc > 2) rng.seed(std::strtoull(argv[2], nullptr, 10));
    for (int i = 0; i < cases; ++i) {
        if (i % 100 == 0) sdhip_set_tuning(("f8_form=" + std::to_string(rng() % 7)).c_str());
        products();
        turns();
        norms();
    }
    std::printf("%d cases: no error\n", cases);
    return 0;
}
