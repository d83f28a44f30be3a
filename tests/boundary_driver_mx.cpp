// Host-side check of include/scmx_mx.h, as boundary_driver.cpp is of scmx.h: built with AddressSanitizer and UBSan on the host pass,
// run on a machine WITHOUT a GPU, every entry point called with null pointers, bad shapes, sizes at the 32-bit limits and seeded random
// integers.  The pointers handed in are not memory (but the host array of scmx_cache4_keep, which is read).
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <random>
#include <vector>

#include "../include/scmx_mx.h"

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

    const auto quantize = [&](const void* x, int type, int64_t ldx, const uint16_t* nw, int M, int K, int shift = 0) {
        return scmx_mx_quantize(x, type, ldx, nw, 1e-6f, p(2) + shift, p(3), M, K, nullptr);
    };
    expect_valid(quantize(p(0), SCMX_MX_BF16, 2048, nullptr, 8192, 2048), "quantize");
    expect_valid(quantize(p(0) + 2, SCMX_MX_F16, 2051, nullptr, 3, 2048), "quantize fp16 at odd places");
    expect_valid(quantize(p(0), SCMX_MX_BF16, 16384, u16(1), 1, 16384), "quantize a norm");
    expect_valid(quantize(p(0), SCMX_MX_F32, 32, nullptr, 2147483647, 32), "quantize, most rows");
    expect_valid(quantize(p(0), SCMX_MX_BF16, 32, u16(1), 2147483647, 32), "quantize a norm, most rows");
    expect_valid(quantize(p(0), SCMX_MX_F32, 1 << 30, nullptr, 1, 1 << 30), "quantize, longest rows");
    expect(quantize(p(0), SCMX_MX_F32, (1 << 30) + 32, nullptr, 1, (1 << 30) + 32), SCMX_ERR_ARG, "quantize, rows too long");
    expect(quantize(nullptr, SCMX_MX_BF16, 32, nullptr, 0, 32), SCMX_OK, "quantize nothing");
    expect(quantize(nullptr, SCMX_MX_BF16, 32, nullptr, 1, 32), SCMX_ERR_ARG, "quantize without rows");
    expect(quantize(p(0), 3, 32, nullptr, 1, 32), SCMX_ERR_ARG, "quantize another type");
    expect(quantize(p(0), SCMX_MX_BF16, 48, nullptr, 1, 48), SCMX_ERR_ARG, "quantize half a block");
    expect(quantize(p(0), SCMX_MX_BF16, 63, nullptr, 2, 64), SCMX_ERR_ARG, "quantize rows that overlap");
    expect(quantize(p(0), SCMX_MX_BF16, INT64_MAX, nullptr, 2, 64), SCMX_ERR_ARG, "quantize rows too far apart");
    expect(quantize(p(0), SCMX_MX_F32, 64, u16(1), 2, 64), SCMX_ERR_ARG, "quantize a norm of float32");
    expect(quantize(p(0), SCMX_MX_BF16, 16416, u16(1), 2, 16416), SCMX_ERR_ARG, "quantize a norm of too many values");
    expect(quantize(p(0) + 1, SCMX_MX_BF16, 64, nullptr, 2, 64), SCMX_ERR_ARG, "quantize misaligned rows");
    expect(quantize(p(0), SCMX_MX_BF16, 64, nullptr, 2, 64, 8), SCMX_ERR_ARG, "quantize to misaligned codes");

    expect_valid(scmx_mx_dequantize(p(0), p(1), p(2), SCMX_MX_F32, 100, 96, nullptr), "dequantize");
    expect(scmx_mx_dequantize(nullptr, nullptr, nullptr, SCMX_MX_BF16, 0, 96, nullptr), SCMX_OK, "dequantize nothing");
    expect(scmx_mx_dequantize(p(0), p(1), p(2), SCMX_MX_F16, 100, 96, nullptr), SCMX_ERR_ARG, "dequantize to fp16");
    expect(scmx_mx_dequantize(p(0), p(1), p(2) + 2, SCMX_MX_BF16, 100, 96, nullptr), SCMX_ERR_ARG, "dequantize misaligned");
    expect(scmx_mx_dequantize(p(0), nullptr, p(2), SCMX_MX_BF16, 100, 96, nullptr), SCMX_ERR_ARG, "dequantize without scales");

    const auto mm = [&](int epi, int M, int N, int K, const uint16_t* res = nullptr, int shift = 0) {
        return scmx_mx_mm(p(0) + shift, p(1), p(2), p(3), res, u16(5), epi, M, N, K, nullptr);
    };
    for (int M : {1, 16, 17, 333, 5000})
        for (int K : {32, 96, 2048, 8192})
            for (int epi : {1, 2, 3}) expect_valid(mm(epi, M, 4096, K, u16(4)), "mm");
    expect_valid(mm(1, 2147483647, 3, 32), "mm, most rows");
    expect_valid(mm(1, 5, 1 << 26, 32), "mm, most columns");
    expect(mm(1, 5, (1 << 26) + 1, 32), SCMX_ERR_ARG, "mm, too many columns");
    expect(mm(1, 2147483647, 15, 64), SCMX_ERR_ARG, "mm, too many rows");
    expect(mm(1, 0, 64, 64), SCMX_OK, "mm of nothing");
    expect(mm(0, 1, 64, 64), SCMX_ERR_ARG, "mm, epilogue 0");
    expect(mm(4, 1, 64, 64), SCMX_ERR_ARG, "mm, epilogue 4");
    expect(mm(1, 1, 64, 48), SCMX_ERR_ARG, "mm, half a block");
    expect(mm(1, 1, 64, (1 << 23) + 32), SCMX_ERR_ARG, "mm, K too long");
    expect(mm(2, 1, 64, 64), SCMX_ERR_ARG, "mm without a residual");
    expect(mm(3, 1, 66, 64), SCMX_ERR_ARG, "mm, SwiGLU of 66 columns");
    expect(mm(1, 1, 64, 64, nullptr, 8), SCMX_ERR_ARG, "mm of misaligned codes");
    expect(mm(1, 2147483647, 2147483647, 32), SCMX_ERR_ARG, "mm, too many results");
    expect(scmx_mx_mm(nullptr, p(1), p(2), p(3), nullptr, u16(5), 1, 1, 64, 64, nullptr), SCMX_ERR_ARG, "mm without rows");

    const auto linear = [&](int epi, int M, int N, int K, int64_t ldx, const uint16_t* nw, size_t bytes, void* work, const uint16_t* x) {
        return scmx_mx_linear(x, ldx, nw, 1e-6f, p(2), p(3), u16(4), u16(5), epi, M, N, K, work, bytes, nullptr);
    };
    expect_valid(linear(1, 1, 4096, 2048, 2048, nullptr, 0, nullptr, u16(0) + 1), "linear of one row");
    expect_valid(linear(3, 100, 4096, 2048, 2051, u16(1), scmx_mx_linear_workspace(100, 4096, 2048, 1), p(6), u16(0)), "linear of a norm");
    expect(linear(1, 0, 4096, 2048, 2048, nullptr, 0, nullptr, nullptr), SCMX_OK, "linear of nothing");
    expect(linear(1, 100, 4096, 2048, 2048, nullptr, scmx_mx_linear_workspace(100, 4096, 2048, 0) - 1, p(6), u16(0)), SCMX_ERR_WORKSPACE, "linear, small workspace");
    expect(linear(1, 1, 4096, 2048, 2048, u16(1), 0, nullptr, u16(0)), SCMX_ERR_WORKSPACE, "linear of a norm without a workspace");
    expect(linear(1, 100, 4096, 2048, 2048, nullptr, size_t(1) << 30, p(6) + 8, u16(0)), SCMX_ERR_WORKSPACE, "linear, misaligned workspace");
    expect(linear(1, 2, 4096, 2048, 2047, nullptr, 0, nullptr, u16(0)), SCMX_ERR_ARG, "linear of rows that overlap");
    expect(linear(1, 2, 4096, 2048, INT64_MAX, nullptr, 0, nullptr, u16(0)), SCMX_ERR_ARG, "linear of rows too far apart");
    expect(linear(1, 2, 4096, 32768, 32768, u16(1), size_t(1) << 30, p(6), u16(0)), SCMX_ERR_ARG, "linear, a norm of too many values");
    if (scmx_mx_linear_workspace(0, 1, 32, 1) || scmx_mx_linear_workspace(1, 0, 32, 1) || scmx_mx_linear_workspace(1, 1, 33, 1) || scmx_mx_linear_workspace(1, 4096, 2048, 0) ||
        scmx_mx_linear_workspace(1, 4096, 2048, 1) != 1024 + 64 || scmx_mx_linear_workspace(333, 64, 96, 1) != 333 * 51 || scmx_mx_linear_workspace(2147483647, 2147483647, 1 << 23, 0) == 0)
        ++failures;

    const auto write = [&](const uint16_t* y, uint8_t* ks, uint8_t* vs, int L, int hq, int hk, int d, int64_t pos, int rows, const int64_t* dev = nullptr) {
        return scmx_cache4_write(nullptr, nullptr, nullptr, y, u16(1), u16(2), 1e-6f, u16(3), p(4), p(5), ks, vs, L, hq, hk, d, f32(8), nullptr, dev, pos, rows, nullptr);
    };
    expect_valid(write(u16(0), p(6), p(7), 4, 16, 8, 128, 60, 64), "cache4_write");
    expect_valid(write(u16(0), p(6), p(7), 4, 16, 8, 128, -9, 64, i64(9)), "cache4_write, position on the device");
    expect(write(nullptr, p(6), p(7), 0, 16, 8, 128, 64, 64), SCMX_OK, "cache4_write of nothing");
    expect(write(nullptr, p(6), p(7), 4, 16, 8, 128, 0, 64), SCMX_ERR_ARG, "cache4_write without input");
    expect(write(u16(0), p(6), nullptr, 4, 16, 8, 128, 0, 64), SCMX_ERR_ARG, "cache4_write with one scale");
    expect(write(u16(0), p(6), p(6), 4, 16, 8, 128, 0, 64), SCMX_ERR_ARG, "cache4_write with both scales in one place");
    expect(write(u16(0), p(6) + 2, p(7), 4, 16, 8, 128, 0, 64), SCMX_ERR_ARG, "cache4_write, misaligned scales");
    expect(write(u16(0), p(6), p(7), 4, 16, 8, 96, 0, 64), SCMX_ERR_ARG, "cache4_write d 96");
    expect(write(u16(0), p(6), p(7), 4, 16, 8, 128, 61, 64), SCMX_ERR_ARG, "cache4_write past the cache");
    expect(write(u16(0), p(6), p(7), 65, 16, 8, 128, 0, 64, i64(9)), SCMX_ERR_ARG, "cache4_write of more rows than the cache has");
    expect(write(u16(0) + 1, p(6), p(7), 4, 16, 8, 128, 0, 64), SCMX_ERR_ARG, "cache4_write misaligned");
    expect(scmx_cache4_write(i32(0), nullptr, f32(1), nullptr, u16(1), u16(2), 1e-6f, u16(3), p(4), p(5), p(6), p(7), 1, 1, 1, 64, f32(8), nullptr, nullptr, 0, 4, nullptr),
           SCMX_ERR_ARG, "cache4_write of accumulators without scales");

    expect_valid(scmx_cache4_read(p(0), p(1), p(2), p(3), u16(4), u16(5), 8, 128, 100, 3, 97, nullptr), "cache4_read");
    expect(scmx_cache4_read(p(0), p(1), p(2), p(3), nullptr, nullptr, 8, 128, 100, 100, 0, nullptr), SCMX_OK, "cache4_read of nothing");
    expect(scmx_cache4_read(p(0), p(1), p(2), p(3), u16(4), u16(5), 8, 128, 100, 4, 97, nullptr), SCMX_ERR_ARG, "cache4_read past the cache");
    expect(scmx_cache4_read(p(0), p(1), nullptr, p(3), u16(4), u16(5), 8, 128, 100, 0, 1, nullptr), SCMX_ERR_ARG, "cache4_read without a scale");

    std::vector<uint64_t> t(4 * 1024);
    for (size_t i = 0; i < t.size(); ++i) t[i] = uint64_t(uintptr_t(p(3))) + 4096 * (i * 1531 % t.size());
    expect_valid(scmx_cache4_keep(t.data(), 1024, 8, 128, 100, i32(0), i32(1), 64, nullptr, 36, nullptr), "cache4_keep, 1024 layers");
    expect_valid(scmx_cache4_keep(t.data(), 28, 8, 256, 100, i32(0), i32(1), 1, i64(2), 0, nullptr), "cache4_keep");
    expect(scmx_cache4_keep(t.data(), 0, 8, 256, 100, i32(0), i32(1), 1, nullptr, 0, nullptr), SCMX_OK, "cache4_keep of no layers");
    expect(scmx_cache4_keep(t.data(), 28, 8, 256, 100, i32(0), i32(1), 65, nullptr, 0, nullptr), SCMX_ERR_ARG, "cache4_keep of 65 rows");
    expect(scmx_cache4_keep(t.data(), 28, 8, 256, 100, i32(0), i32(1), 64, nullptr, 37, nullptr), SCMX_ERR_ARG, "cache4_keep past the cache");
    for (uint64_t bad : {uint64_t(0), t[6], t[6] + 4}) {
        const uint64_t good = t[7];
        t[7] = bad;
        expect(scmx_cache4_keep(t.data(), 28, 8, 256, 100, i32(0), i32(1), 4, nullptr, 0, nullptr), SCMX_ERR_ARG, "cache4_keep with a null, repeated or misaligned layer");
        t[7] = good;
    }

    const auto attend = [&](int T, int hq, int hk, int d, int rows, int64_t pos, float scale, float* work, int splits, const uint8_t* vs) {
        return scmx_attn_tree4(u16(0), p(1), p(2), p(6), vs, i64(3), nullptr, pos, u16(4), T, hq, hk, d, rows, scale, work, splits, nullptr);
    };
    expect_valid(attend(64, 32, 8, 128, 100, 36, 0.1f, f32(5), 64, p(7)), "attn_tree4");
    expect_valid(attend(1, 16, 4, 256, 100, 0, -0.1f, nullptr, 1, p(7)), "attn_tree4, one token");
    expect_valid(attend(64, 4096, 1, 64, 2147483647, 2147483583, 0.1f, f32(5), 64, p(7)), "attn_tree4 at the limits");
    expect(attend(65, 32, 8, 128, 100, 0, 0.1f, nullptr, 1, p(7)), SCMX_ERR_ARG, "attn_tree4 of 65 nodes");
    expect(attend(4, 32, 8, 128, 100, 97, 0.1f, nullptr, 1, p(7)), SCMX_ERR_ARG, "attn_tree4 past the cache");
    expect(attend(4, 32, 7, 128, 100, 0, 0.1f, nullptr, 1, p(7)), SCMX_ERR_ARG, "attn_tree4, uneven heads");
    expect(attend(4, 4097, 1, 128, 100, 0, 0.1f, nullptr, 1, p(7)), SCMX_ERR_ARG, "attn_tree4, 4097 heads a KV head");
    expect(attend(4, 32, 8, 128, 100, 0, 0.1f, nullptr, 2, p(7)), SCMX_ERR_ARG, "attn_tree4, splits without a workspace");
    expect(attend(4, 32, 8, 128, 100, 0, 0.1f, f32(5), 65, p(7)), SCMX_ERR_ARG, "attn_tree4, 65 splits");
    expect(attend(4, 32, 8, 128, 100, 0, __builtin_nanf(""), nullptr, 1, p(7)), SCMX_ERR_ARG, "attn_tree4, scale NaN");
    expect(attend(4, 32, 8, 128, 100, 0, 3e38f, nullptr, 1, p(7)), SCMX_ERR_ARG, "attn_tree4, scale past float32 in powers of two");
    expect(attend(4, 32, 8, 128, 100, 0, 0.1f, nullptr, 1, nullptr), SCMX_ERR_ARG, "attn_tree4 with one scale");
    expect(attend(4, 32, 8, 128, 100, 0, 0.1f, nullptr, 1, p(7) + 2), SCMX_ERR_ARG, "attn_tree4, misaligned scales");
    if (scmx_attn_tree4_splits(65, 100, 8, 8, 128) != 1 || scmx_attn_tree4_splits(1, 2147483647, 65535, 65535, 64) != 1 || scmx_attn_tree4_splits(1, 100000, 16, 8, 128) != 64) ++failures;

    std::mt19937 rng(78);
    const int special[] = {0, 1, -1, 2, 63, 64, 65, 128, 256, 65535, 65536, 2147483647, -2147483647 - 1, 2147483583, 4096, 1 << 30};
    const auto r = [&]() { return rng() % 3 ? special[rng() % (sizeof special / sizeof *special)] : int(rng()); };
    const auto dim = [&]() { const int d[] = {64, 128, 256}; return rng() % 4 ? d[rng() % 3] : r(); };
    const auto small = [&]() { return rng() % 2 ? int(rng() % 70) : r(); };
    const auto block = [&]() { return rng() % 4 ? 32 * int(1 + rng() % 300) : r(); };
    const auto maybe = [&](uint16_t* x) { return rng() % 2 ? x : nullptr; };
    for (int i = 0; i < 4000; ++i) {
        const int64_t* dev = rng() % 2 ? i64(9) : nullptr;
        const int64_t pos = int64_t(r()) * (rng() % 3);
        expect_status(quantize(p(0), int(rng() % 4), int64_t(r()) * (rng() % 4), maybe(u16(1)), r(), block()), "fuzz quantize");
        expect_status(scmx_mx_dequantize(p(0), p(1), p(2), int(rng() % 4), r(), block(), nullptr), "fuzz dequantize");
        expect_status(mm(int(rng() % 5), r(), r(), block(), maybe(u16(4))), "fuzz mm");
        const int M = r(), N = r(), K = block();
        uint16_t* const nw = maybe(u16(1));
        expect_status(linear(int(rng() % 5), M, N, K, rng() % 4 ? K : r(), nw, rng() % 4 ? scmx_mx_linear_workspace(M, N, K, nw != nullptr) : size_t(r()), p(6), u16(0)), "fuzz linear");
        expect_status(scmx_cache4_write(rng() % 4 ? nullptr : i32(0), rng() % 2 ? f32(1) : nullptr, rng() % 2 ? f32(2) : nullptr, u16(0), u16(1), u16(2), 1e-6f, u16(3), p(4),
                                        p(5), p(6), p(7), small(), small(), small(), dim(), f32(8), rng() % 2 ? i32(9) : nullptr, dev, pos, r(), nullptr),
                      "fuzz cache4_write");
        expect_status(scmx_cache4_read(p(0), p(1), p(2), p(3), u16(4), u16(5), small(), dim(), r(), r(), r(), nullptr), "fuzz cache4_read");
        expect_status(scmx_cache4_keep(t.data(), int(rng() % 1030), small(), dim(), r(), i32(0), i32(1), small(), dev, pos, nullptr), "fuzz cache4_keep");
        expect_status(scmx_attn_tree4(u16(0), p(1), p(2), p(6), p(7), rng() % 2 ? i64(3) : nullptr, dev, pos, u16(4), small(), small(), small(), dim(), r(), 0.1f,
                                      rng() % 2 ? f32(5) : nullptr, small(), nullptr),
                      "fuzz attn_tree4");
        const int s = scmx_attn_tree4_splits(small(), r(), small(), small(), dim());
        if (s < 1 || s > 64) ++failures;
    }
    printf("%ld calls, %d failure(s)\n", calls, failures);
    return failures ? 1 : 0;
}
