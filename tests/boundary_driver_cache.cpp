// Host-side check of include/scmx_cache.h, as boundary_driver.cpp is of scmx.h: built with AddressSanitizer and UBSan on the host pass,
// run on a machine WITHOUT a GPU, every entry point called with null pointers, bad shapes, sizes at the 32-bit limits and seeded random
// integers.  The pointers handed in are not memory (but the host array of scmx_cache_keep, which is read).
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <random>
#include <vector>

#include "../include/scmx_cache.h"

extern "C" int hipGetDeviceCount(int* count);

static int failures = 0;
static long calls = 0;

static void expect(int rc, int want, const char* what) {
    ++calls;
    if (rc != want) {
        printf("FAIL %s: status %d, expected %d (%s)\n", what, rc, want, scmx_last_error());
        ++failures;
    }
}
static void expect_valid(int rc, const char* what) {   // ends at the launch here, or has nothing to do
    ++calls;
    if (rc != SCMX_OK && rc != SCMX_ERR_LAUNCH) {
        printf("FAIL %s: plausible arguments refused with %d (%s)\n", what, rc, scmx_last_error());
        ++failures;
    }
}
static void expect_status(int rc, const char* what) {
    ++calls;
    if (rc > 0 || rc < SCMX_ERR_WORKSPACE) {
        printf("FAIL %s: undocumented status %d\n", what, rc);
        ++failures;
    }
    if (rc != SCMX_OK && !scmx_last_error()[0]) {
        printf("FAIL %s: status %d without a message\n", what, rc);
        ++failures;
    }
}

int main() {
    int devices = 0;
    if (hipGetDeviceCount(&devices) == 0 && devices > 0) {
        printf("a GPU is present: this check passes addresses that are not memory and is meant for machines without one\n");
        return 77;
    }
    uint8_t* const P = reinterpret_cast<uint8_t*>(uintptr_t(0x7100000000ull));
    const auto p = [&](int i) { return P + size_t(i) * (size_t(1) << 30); };
    const auto u16 = [&](int i) { return reinterpret_cast<uint16_t*>(p(i)); };
    const auto f32 = [&](int i) { return reinterpret_cast<float*>(p(i)); };
    const auto i32 = [&](int i) { return reinterpret_cast<int32_t*>(p(i)); };
    const auto i64 = [&](int i) { return reinterpret_cast<int64_t*>(p(i)); };
    const auto i8 = [&](int i) { return reinterpret_cast<int8_t*>(p(i)); };

    expect(scmx_cache_write(nullptr, nullptr, nullptr, u16(0), u16(1), u16(2), 1e-6f, u16(3), p(4), p(4), nullptr, nullptr, 1, 4, 2, 64, f32(8), nullptr, nullptr, 0, 16, nullptr),
           SCMX_ERR_ARG, "write: keys and values in one cache");
    const auto write = [&](const uint16_t* y, float* ks, float* vs, int L, int hq, int hk, int d, int64_t pos, int rows, const int64_t* dev = nullptr) {
        return scmx_cache_write(nullptr, nullptr, nullptr, y, u16(1), u16(2), 1e-6f, u16(3), p(4), p(5), ks, vs, L, hq, hk, d, f32(8), nullptr, dev, pos, rows, nullptr);
    };
    expect_valid(write(u16(0), nullptr, nullptr, 4, 16, 8, 128, 10, 64), "cache_write bf16");
    expect_valid(write(u16(0), f32(6), f32(7), 4, 16, 8, 128, 60, 64), "cache_write 8 bits");
    expect_valid(write(u16(0), f32(6), f32(7), 4, 16, 8, 128, -9, 64, i64(9)), "cache_write, position on the device");
    expect(write(nullptr, f32(6), f32(7), 0, 16, 8, 128, 64, 64), SCMX_OK, "cache_write of nothing");
    expect(write(nullptr, f32(6), f32(7), 4, 16, 8, 128, 0, 64), SCMX_ERR_ARG, "cache_write without input");
    expect(write(u16(0), f32(6), nullptr, 4, 16, 8, 128, 0, 64), SCMX_ERR_ARG, "cache_write with one scale");
    expect(write(u16(0), nullptr, nullptr, 4, 16, 8, 96, 0, 64), SCMX_ERR_ARG, "cache_write d 96");
    expect(write(u16(0), nullptr, nullptr, 4, 16, 8, 128, 61, 64), SCMX_ERR_ARG, "cache_write past the cache");
    expect(write(u16(0), nullptr, nullptr, 65, 16, 8, 128, 0, 64, i64(9)), SCMX_ERR_ARG, "cache_write of more rows than the cache has");
    expect(write(u16(0) + 1, nullptr, nullptr, 4, 16, 8, 128, 0, 64), SCMX_ERR_ARG, "cache_write misaligned");
    expect(scmx_cache_write(i32(0), nullptr, f32(1), nullptr, u16(1), u16(2), 1e-6f, u16(3), p(4), p(5), nullptr, nullptr, 1, 1, 1, 64, f32(8), nullptr, nullptr, 0, 4, nullptr),
           SCMX_ERR_ARG, "cache_write of accumulators without scales");

    expect_valid(scmx_cache_read(i8(0), i8(1), f32(2), f32(3), u16(4), u16(5), 8, 128, 100, 3, 97, nullptr), "cache_read");
    expect(scmx_cache_read(i8(0), i8(1), f32(2), f32(3), nullptr, nullptr, 8, 128, 100, 100, 0, nullptr), SCMX_OK, "cache_read of nothing");
    expect(scmx_cache_read(i8(0), i8(1), f32(2), f32(3), u16(4), u16(5), 8, 128, 100, 4, 97, nullptr), SCMX_ERR_ARG, "cache_read past the cache");
    expect(scmx_cache_read(i8(0), i8(1), nullptr, f32(3), u16(4), u16(5), 8, 128, 100, 0, 1, nullptr), SCMX_ERR_ARG, "cache_read without a scale");

    std::vector<uint64_t> t(4 * 1024);
    for (size_t i = 0; i < t.size(); ++i) t[i] = uint64_t(uintptr_t(p(3))) + 4096 * (i * 1531 % t.size());
    expect_valid(scmx_cache_keep(t.data(), 1024, 1, 8, 128, 100, i32(0), i32(1), 64, nullptr, 36, nullptr), "cache_keep, 1024 layers");
    expect_valid(scmx_cache_keep(t.data(), 28, 0, 8, 256, 100, i32(0), i32(1), 1, i64(2), 0, nullptr), "cache_keep");
    expect(scmx_cache_keep(t.data(), 0, 0, 8, 256, 100, i32(0), i32(1), 1, nullptr, 0, nullptr), SCMX_OK, "cache_keep of no layers");
    expect(scmx_cache_keep(t.data(), 28, 0, 8, 256, 100, i32(0), i32(1), 65, nullptr, 0, nullptr), SCMX_ERR_ARG, "cache_keep of 65 rows");
    expect(scmx_cache_keep(t.data(), 28, 0, 8, 256, 100, i32(0), i32(1), 64, nullptr, 37, nullptr), SCMX_ERR_ARG, "cache_keep past the cache");
    t[7] = 0;
    expect(scmx_cache_keep(t.data(), 28, 0, 8, 256, 100, i32(0), i32(1), 4, nullptr, 0, nullptr), SCMX_ERR_ARG, "cache_keep with a null layer");
    t[7] = t[6];
    expect(scmx_cache_keep(t.data(), 28, 0, 8, 256, 100, i32(0), i32(1), 4, nullptr, 0, nullptr), SCMX_ERR_ARG, "cache_keep with a cache twice");
    t[7] = t[6] + 4;
    expect(scmx_cache_keep(t.data(), 28, 0, 8, 256, 100, i32(0), i32(1), 4, nullptr, 0, nullptr), SCMX_ERR_ARG, "cache_keep with a misaligned layer");
    t[7] = uint64_t(uintptr_t(p(3))) + 4096 * (7 * 1531 % t.size());

    const auto attend = [&](int T, int hq, int hk, int d, int rows, int64_t pos, float scale, float* work, int splits, float* ks = nullptr, float* vs = nullptr) {
        return scmx_attn_tree(u16(0), p(1), p(2), ks, vs, i64(3), nullptr, pos, u16(4), T, hq, hk, d, rows, scale, work, splits, nullptr);
    };
    expect_valid(attend(64, 32, 8, 128, 100, 36, 0.1f, f32(5), 64), "attn_tree");
    expect_valid(attend(1, 16, 4, 256, 100, 0, -0.1f, nullptr, 1, f32(6), f32(7)), "attn_tree, one token, 8 bits");
    expect_valid(attend(64, 4096, 1, 64, 2147483647, 2147483583, 0.1f, f32(5), 64), "attn_tree at the limits");
    expect(attend(65, 32, 8, 128, 100, 0, 0.1f, nullptr, 1), SCMX_ERR_ARG, "attn_tree of 65 nodes");
    expect(attend(4, 32, 8, 128, 100, 97, 0.1f, nullptr, 1), SCMX_ERR_ARG, "attn_tree past the cache");
    expect(attend(4, 32, 7, 128, 100, 0, 0.1f, nullptr, 1), SCMX_ERR_ARG, "attn_tree, uneven heads");
    expect(attend(4, 4097, 1, 128, 100, 0, 0.1f, nullptr, 1), SCMX_ERR_ARG, "attn_tree, 4097 heads a KV head");
    expect(attend(4, 32, 8, 128, 100, 0, 0.1f, nullptr, 2), SCMX_ERR_ARG, "attn_tree, splits without a workspace");
    expect(attend(4, 32, 8, 128, 100, 0, 0.1f, f32(5), 65), SCMX_ERR_ARG, "attn_tree, 65 splits");
    expect(attend(4, 32, 8, 128, 100, 0, __builtin_nanf(""), nullptr, 1), SCMX_ERR_ARG, "attn_tree, scale NaN");
    expect(attend(4, 32, 8, 128, 100, 0, 0.1f, nullptr, 1, f32(6)), SCMX_ERR_ARG, "attn_tree with one scale");

    const auto verify = [&](const float* draft, double temperature, const float* u, int T, int V, int siblings, void* work, size_t bytes) {
        return scmx_verify_drafts(i64(0), i32(1), p(2), 0, draft, temperature, u, i32(3), i32(4), i64(5), T, V, siblings, work, bytes, nullptr);
    };
    expect_valid(verify(nullptr, 0.0, nullptr, 64, 4194304, 0, p(6), scmx_verify_workspace(64, 4194304, 0)), "verify_drafts, greedy");
    expect_valid(verify(f32(7), 1.0, f32(8), 8, 151936, 16, p(6), scmx_verify_workspace(8, 151936, 16)), "verify_drafts with a draft");
    expect(verify(f32(7), 1.0, f32(8), 8, 151936, 2, p(6), scmx_verify_workspace(8, 151936, 1)), SCMX_ERR_WORKSPACE, "verify_drafts, small workspace");
    expect(verify(f32(7), 1.0, f32(8), 8, 151936, 17, p(6), size_t(1) << 30), SCMX_ERR_ARG, "verify_drafts, 17 siblings");
    expect(verify(nullptr, 1.0, nullptr, 8, 100, 0, p(6), 4096), SCMX_ERR_ARG, "verify_drafts without random numbers");
    expect(verify(nullptr, -1.0, f32(8), 8, 100, 0, p(6), 4096), SCMX_ERR_ARG, "verify_drafts, temperature -1");
    expect(verify(nullptr, 1.0, f32(8), 65, 100, 0, p(6), 4096), SCMX_ERR_ARG, "verify_drafts of 65 nodes");
    expect(verify(nullptr, 1.0, f32(8), 1, 4194305, 0, p(6), size_t(1) << 30), SCMX_ERR_ARG, "verify_drafts, vocabulary");
    if (scmx_attn_tree_splits(65, 100, 8, 8, 128) != 1 || scmx_attn_tree_splits(1, 2147483647, 65535, 65535, 64) != 1) ++failures;
    if (scmx_verify_workspace(65, 100, 0) || scmx_verify_workspace(1, 0, 0) || scmx_verify_workspace(1, 100, 17) || !scmx_verify_workspace(1, 1, 0)) ++failures;

    std::mt19937 rng(77);
    const int special[] = {0, 1, -1, 2, 63, 64, 65, 128, 256, 65535, 65536, 2147483647, -2147483647 - 1, 2147483583, 4096, 1 << 30};
    const auto r = [&]() { return rng() % 3 ? special[rng() % (sizeof special / sizeof *special)] : int(rng()); };
    const auto dim = [&]() { const int d[] = {64, 128, 256}; return rng() % 4 ? d[rng() % 3] : r(); };
    const auto small = [&]() { return rng() % 2 ? int(rng() % 70) : r(); };
    const auto maybe = [&](float* x) { return rng() % 2 ? x : nullptr; };
    for (int i = 0; i < 4000; ++i) {
        const int64_t* dev = rng() % 2 ? i64(9) : nullptr;
        const int64_t pos = int64_t(r()) * (rng() % 3);
        expect_status(scmx_cache_write(rng() % 4 ? nullptr : i32(0), maybe(f32(1)), maybe(f32(2)), u16(0), u16(1), u16(2), 1e-6f, u16(3), p(4), p(5), maybe(f32(6)), maybe(f32(7)),
                                       small(), small(), small(), dim(), f32(8), rng() % 2 ? i32(9) : nullptr, dev, pos, r(), nullptr),
                      "fuzz cache_write");
        expect_status(scmx_cache_read(i8(0), i8(1), f32(2), f32(3), u16(4), u16(5), small(), dim(), r(), r(), r(), nullptr), "fuzz cache_read");
        expect_status(scmx_cache_keep(t.data(), int(rng() % 1030), int(rng() % 2), small(), dim(), r(), i32(0), i32(1), small(), dev, pos, nullptr), "fuzz cache_keep");
        expect_status(scmx_attn_tree(u16(0), p(1), p(2), maybe(f32(6)), maybe(f32(7)), rng() % 2 ? i64(3) : nullptr, dev, pos, u16(4), small(), small(), small(), dim(), r(), 0.1f,
                                     maybe(f32(5)), small(), nullptr),
                      "fuzz attn_tree");
        {
            const int s = scmx_attn_tree_splits(small(), r(), small(), small(), dim());
            if (s < 1 || s > 64) ++failures;
        }
        const int T = small(), V = r(), s = int(rng() % 20);
        expect_status(scmx_verify_drafts(i64(0), i32(1), p(2), int(rng() % 2), maybe(f32(7)), rng() % 2 ? 0.0 : 0.7, maybe(f32(8)), i32(3), i32(4), i64(5), T, V, s, p(6),
                                         rng() % 2 ? scmx_verify_workspace(T, V, s) : size_t(r()), nullptr),
                      "fuzz verify_drafts");
    }
    printf("%ld calls, %d failure(s)\n", calls, failures);
    return failures ? 1 : 0;
}
