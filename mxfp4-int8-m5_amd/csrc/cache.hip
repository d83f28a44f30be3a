// A KV cache in bf16 or 8 bits: the append of new tokens (norm, rotary embedding, quantisation in one pass), the read-back for a
// prompt's attention, and the accepted rows of a tree of drafts moved together (include/scmx_cache.h).
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "../../include/scmx_cache.h"
#include "scmx_common.h"

namespace scmx {

constexpr int CNT = 256;
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(4)));

struct WriteArgs {
    const int32_t* acc;
    const float* xscale;
    const float* wscale;
    const uint16_t* y;
    const uint16_t* qn;
    const uint16_t* kn;
    float eps;
    uint16_t* q;
    void* cache[2];      // K, V
    float* scale[2];     // NULL: bf16
    int L, hq, hk;
    const float* inv_freq;
    const int32_t* depth;
    const int64_t* pos_dev;
    int64_t pos0;
    int rows;
};

// Operations over the LPH lanes of a head (8, 16 or 32, aligned), within rows of 16 lanes by row operations: through LDS (shuffles) a
// head took twenty trips of a hundred cycles, one after the other.
template <int CTRL>
__device__ __forceinline__ float row_op(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int LPH, typename F>
__device__ __forceinline__ float over_head(float v, F&& f) {   // f of all lanes' values, in every lane
    v = f(v, row_op<0xB1>(v));    // quad_perm 1 0 3 2
    v = f(v, row_op<0x4E>(v));    // quad_perm 2 3 0 1
    v = f(v, row_op<0x141>(v));   // row_half_mirror: the other quad of eight
    if (LPH >= 16) v = f(v, row_op<0x140>(v));   // row_mirror: the other eight of sixteen
    if (LPH >= 32) v = f(v, __shfl_xor(v, 16, WAVE));
    return v;
}
template <int LPH>
__device__ __forceinline__ float partner(float v) {   // of the lane half a head away
    if (LPH == 8) return row_op<0x1B>(row_op<0x141>(v));   // 7 - j, then its quad reversed: j ^ 4
    if (LPH == 16) return row_op<0x128>(v);                // row_ror 8
    return __shfl_xor(v, 16, WAVE);
}

// One token per blockIdx.x.  A head of D values is held by D / 8 lanes, eight consecutive values each: 16-byte loads, 16-byte
// (bf16) or 8-byte (codes) stores, the norm's sum and the row's maximum over the lanes of the group, and the partner of a
// rotation half a group away at the same place.  Per head (x: the row, n: its norm)
//     n = x / sqrt(mean(x^2) + eps) * w,  (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * inv_freq
// The angle is formed and reduced to one turn in float64: in float32 a position of 100000 is off by 4e-3 of a radian, as much as
// the result's rounding.  Everything else is float32 and rounded once, to bf16 or to a code.
// Bound by memory for a prompt (the next head's row is requested before this one's is worked on), by latency (the row, then two
// chains of cross-lane sums) for a few tokens.  8 bits: 16 tokens of 16:8 x 128 3.2 us, 2501 of 32:8 x 128 12.7 (4.4 TB/s), from
// accumulators (twice the bytes to read) 3.3 and 21.8 in a graph (16.2 from bf16 there; 4.0 TB/s).
template <int D, bool EIGHT, bool ACC>
__global__ __launch_bounds__(CNT) void cache_write_kernel(const WriteArgs a) {
    constexpr int LPH = D / 8, GROUPS = CNT / LPH;
    __shared__ float s_sin[D / 2], s_cos[D / 2];
    const int row = blockIdx.x, grp = threadIdx.x / LPH, j = threadIdx.x % LPH;
    const int heads = a.hq + 2 * a.hk, stride = gridDim.y * GROUPS;
    const int64_t pos = a.pos_dev ? a.pos_dev[0] : a.pos0;
    const bool fits = pos >= 0 && pos <= int64_t(a.rows) - a.L;
    // the lane's values of a head as they come, and as numbers
    struct Raw {
        u32x4 w[ACC ? 2 : 1];
    };
    const auto load = [&](int g, Raw& r) {
        const size_t at = (size_t(row) * heads + g) * D + 8 * j;
        if constexpr (ACC) {
            r.w[0] = *reinterpret_cast<const u32x4u*>(a.acc + at);
            r.w[1] = *reinterpret_cast<const u32x4u*>(a.acc + at + 4);
        } else {
            r.w[0] = *reinterpret_cast<const u32x4*>(a.y + at);
        }
    };
    Raw raw;
    int g = blockIdx.y * GROUPS + grp;
    if (g < heads) load(g, raw);   // on its way beside the angles
    const u32x4 wq = *reinterpret_cast<const u32x4*>(a.qn + 8 * j), wk = *reinterpret_cast<const u32x4*>(a.kn + 8 * j);
    if (threadIdx.x < D / 2) {
        const double turns = double(pos + (a.depth ? a.depth[row] : row)) * double(a.inv_freq[threadIdx.x]) * 0.15915494309189535;
        sincospif(float(2.0 * (turns - rint(turns))), &s_sin[threadIdx.x], &s_cos[threadIdx.x]);
    }
    __syncthreads();
    for (; g < heads; g += stride) {   // (a group is whole or absent)
        float x[8];
        if constexpr (ACC) {
            const float xs = a.xscale[row];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[i] = round_bf16(__fmul_rn(__fmul_rn(float(int32_t(raw.w[i / 4][i % 4])), xs), a.wscale[g * D + 8 * j + i]));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = bf16_lo(raw.w[0][i]);
                x[2 * i + 1] = bf16_hi(raw.w[0][i]);
            }
        }
        if (g + stride < heads) load(g + stride, raw);
        const bool is_v = g >= a.hq + a.hk;
        if (!is_v) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
            ss = over_head<LPH>(ss, [](float p, float q) { return p + q; });
            const float inv = __fdiv_rn(1.0f, sqrtf(__fdiv_rn(ss, float(D)) + a.eps));
            const u32x4 w = g < a.hq ? wq : wk;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = x[2 * i] * inv * bf16_lo(w[i]);
                x[2 * i + 1] = x[2 * i + 1] * inv * bf16_hi(w[i]);
            }
            const int at = 8 * (j % (LPH / 2));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float other = partner<LPH>(x[i]) * s_sin[at + i];
                x[i] = __builtin_fmaf(x[i], s_cos[at + i], j < LPH / 2 ? -other : other);
            }
        }
        if (g >= a.hq && !fits) continue;
        const int which = is_v, h = g - a.hq - (is_v ? a.hk : 0);
        const size_t at = g < a.hq ? size_t(row) * a.hq + g : size_t(h) * a.rows + size_t(pos) + row;   // in rows of D
        if (EIGHT && g >= a.hq) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]) <= 3.4028234e38f ? fabsf(x[i]) : __builtin_inff());   // (NaN too)
            top = over_head<LPH>(top, [](float p, float q) { return fmaxf(p, q); });
            const bool finite = top < __builtin_inff(), any = finite && top >= 0x1p-100f;
            const float inv = any ? __fdiv_rn(127.0f, top) : 0.0f;
            u32x2 w = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (any) w[i / 4] |= (uint32_t(quant_code(x[i], inv)) & 0xFFu) << (8 * (i % 4));
            *reinterpret_cast<u32x2*>(static_cast<int8_t*>(a.cache[which]) + at * D + 8 * j) = w;
            if (j == 0) a.scale[which][at] = any ? __fdiv_rn(top, 127.0f) : finite ? 0.0f : __builtin_nanf("");
        } else {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = f32_to_bf16x2(x[2 * i], x[2 * i + 1]);
            uint16_t* dst = g < a.hq ? a.q : static_cast<uint16_t*>(a.cache[which]);
            *reinterpret_cast<u32x4*>(dst + at * D + 8 * j) = w;
        }
    }
}

// 16 codes a lane, blockIdx.y: KV head, blockIdx.z: K or V.  A byte read for two written, but a thread has a single load in flight:
// 2501 rows of 8 x 128 5.0 us, 3.1 TB/s.
template <int D>
__global__ __launch_bounds__(CNT) void cache_read_kernel(const int8_t* kc, const int8_t* vc, const float* ks, const float* vs, uint16_t* k,
                                                         uint16_t* v, int rows, int row0, int n) {
    const int8_t* codes = (blockIdx.z ? vc : kc) + (size_t(blockIdx.y) * rows + row0) * D;
    const float* scales = (blockIdx.z ? vs : ks) + size_t(blockIdx.y) * rows + row0;
    uint16_t* out = (blockIdx.z ? v : k) + size_t(blockIdx.y) * n * D;
    const size_t at = (size_t(blockIdx.x) * CNT + threadIdx.x) * 16;
    if (at >= size_t(n) * D) return;
    const u32x4 c = *reinterpret_cast<const u32x4*>(codes + at);
    const float s = scales[at / D];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t two = c[2 * h + i / 2] >> (16 * (i % 2));
            w[i] = f32_to_bf16x2(float(int8_t(two)) * s, float(int8_t(two >> 8)) * s);
        }
        *reinterpret_cast<u32x4*>(out + at + 8 * h) = w;
    }
}

// The layers of one launch: their pointers travel in the kernel's arguments.
constexpr int KEEP_LAYERS = 32;
struct KeepArgs {
    void* t[KEEP_LAYERS][4];
};

// blockIdx.x: KV head, y: K or V, z: layer.  The rows are read whole before any is written (a row may be both); up to 64 rows of up
// to 512 bytes.  Bound by latency: count, path, rows, stores.
template <int ROWB>
__global__ __launch_bounds__(CNT) void cache_keep_kernel(const KeepArgs a, bool eight, int rows, const int32_t* path, const int32_t* count,
                                                         int T, const int64_t* pos_dev, int64_t pos0) {
    const int64_t pos = pos_dev ? pos_dev[0] : pos0;
    if (pos < 0 || pos > int64_t(rows) - T) return;
    const int kept = min(max(count[0], 0), T);
    const size_t first = size_t(blockIdx.x) * rows + size_t(pos);
    uint8_t* t = static_cast<uint8_t*>(a.t[blockIdx.z][blockIdx.y]) + first * ROWB;
    constexpr int PER = ROWB / 16, N = 64 * PER / CNT;   // 16-byte pieces a row, and a thread
    u32x4 w[N];
    int from[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = threadIdx.x + CNT * i, to = c / PER;
        from[i] = to < kept ? path[to] : -1;
        if (from[i] < 0 || from[i] >= T || from[i] == to) from[i] = -1;
        if (from[i] >= 0) w[i] = *reinterpret_cast<const u32x4*>(t + size_t(from[i]) * ROWB + c % PER * 16);
    }
    float* s = eight ? static_cast<float*>(a.t[blockIdx.z][2 + blockIdx.y]) + first : nullptr;
    const int mine = eight && int(threadIdx.x) < kept ? path[threadIdx.x] : -1;
    const bool moves = mine >= 0 && mine < T;
    float scale = 0.0f;
    if (moves) scale = s[mine];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = threadIdx.x + CNT * i;
        if (from[i] >= 0) *reinterpret_cast<u32x4*>(t + size_t(c / PER) * ROWB + c % PER * 16) = w[i];
    }
    if (moves) s[threadIdx.x] = scale;
}

}  // namespace scmx

using namespace scmx;

// What every entry point on a cache checks: head counts, head dim, rows, and where the rows pos .. pos + n - 1 are.
static int check_cache(const char* who, int hq, int hk, int d, int rows, int64_t n, const int64_t* pos_dev, int64_t pos0) {
    if (hq < 1 || hk < 1 || hq > 65535 || hk > 65535 || rows < 1) {
        set_error("%s: bad head counts or cache size (hq=%d hk=%d rows=%d)", who, hq, hk, rows);
        return SCMX_ERR_ARG;
    }
    if (d != 64 && d != 128 && d != 256) {
        set_error("%s: head dim must be 64, 128 or 256 (d=%d)", who, d);
        return SCMX_ERR_ARG;
    }
    if (n < 0 || n > rows || (!pos_dev && (pos0 < 0 || pos0 > rows - n))) {
        set_error("%s: %lld rows from %lld on do not fit a cache of %d rows", who, (long long)n, (long long)pos0, rows);
        return SCMX_ERR_ARG;
    }
    return SCMX_OK;
}

extern "C" int scmx_cache_write(const int32_t* acc, const float* xscale, const float* wscale, const uint16_t* y, const uint16_t* qn,
                                const uint16_t* kn, float eps, uint16_t* q, void* kcache, void* vcache, float* kscale, float* vscale, int L,
                                int hq, int hk, int d, const float* inv_freq, const int32_t* depth, const int64_t* pos_dev, int64_t pos0,
                                int cache_rows, void* stream) {
    if ((L && ((!acc && !y) || !q)) || (acc && (!xscale || !wscale)) || !qn || !kn || !kcache || !vcache || !inv_freq ||
        !kscale != !vscale) {
        set_error("cache_write: null pointer argument (an 8-bit cache has both scales, a bf16 one none)");
        return SCMX_ERR_ARG;
    }
    if (int rc = check_cache("cache_write", hq, hk, d, cache_rows, L, pos_dev, pos0)) return rc;
    if ((uintptr_t(acc ? nullptr : y) | uintptr_t(qn) | uintptr_t(kn) | uintptr_t(q) | uintptr_t(kcache) | uintptr_t(vcache)) % 16) {
        set_error("cache_write: y, qn, kn, q and the caches must be 16-byte aligned");
        return SCMX_ERR_ARG;
    }
    if (kcache == vcache || (kscale && kscale == vscale)) {
        set_error("cache_write: K and V are one cache");
        return SCMX_ERR_ARG;
    }
    if (L == 0) return SCMX_OK;
    const WriteArgs a{acc, xscale, wscale, y, qn, kn, eps, q, {kcache, vcache}, {kscale, vscale}, L, hq, hk, inv_freq, depth, pos_dev, pos0,
                      cache_rows};
    const int groups = CNT / (d / 8), turns = (hq + 2 * hk + groups - 1) / groups;
    // a few tokens are spread over the CUs; a prompt fills them with a workgroup a token, which then takes the angles once
    const dim3 grid(L, L >= 256 ? 1 : turns);
    const hipStream_t st = (hipStream_t)stream;
    const auto go = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        if (acc && kscale) cache_write_kernel<D, true, true><<<grid, dim3(CNT), 0, st>>>(a);
        else if (acc) cache_write_kernel<D, false, true><<<grid, dim3(CNT), 0, st>>>(a);
        else if (kscale) cache_write_kernel<D, true, false><<<grid, dim3(CNT), 0, st>>>(a);
        else cache_write_kernel<D, false, false><<<grid, dim3(CNT), 0, st>>>(a);
    };
    if (d == 64) go(std::integral_constant<int, 64>{});
    else if (d == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
    return check_launch("cache_write");
}

extern "C" int scmx_cache_read(const int8_t* kcache, const int8_t* vcache, const float* kscale, const float* vscale, uint16_t* k,
                               uint16_t* v, int hk, int d, int cache_rows, int row0, int n, void* stream) {
    if (!kcache || !vcache || !kscale || !vscale || (n && (!k || !v))) {
        set_error("cache_read: null pointer argument");
        return SCMX_ERR_ARG;
    }
    if (int rc = check_cache("cache_read", 1, hk, d, cache_rows, n, nullptr, row0)) return rc;
    if ((uintptr_t(kcache) | uintptr_t(vcache) | uintptr_t(k) | uintptr_t(v)) % 16) {
        set_error("cache_read: the caches and outputs must be 16-byte aligned");
        return SCMX_ERR_ARG;
    }
    if (n == 0) return SCMX_OK;
    const dim3 grid(unsigned((size_t(n) * d / 16 + CNT - 1) / CNT), hk, 2);
    const hipStream_t st = (hipStream_t)stream;
    if (d == 64) cache_read_kernel<64><<<grid, dim3(CNT), 0, st>>>(kcache, vcache, kscale, vscale, k, v, cache_rows, row0, n);
    else if (d == 128) cache_read_kernel<128><<<grid, dim3(CNT), 0, st>>>(kcache, vcache, kscale, vscale, k, v, cache_rows, row0, n);
    else cache_read_kernel<256><<<grid, dim3(CNT), 0, st>>>(kcache, vcache, kscale, vscale, k, v, cache_rows, row0, n);
    return check_launch("cache_read");
}

extern "C" int scmx_cache_keep(const uint64_t* caches, int layers, int eight, int hk, int d, int cache_rows, const int32_t* path,
                               const int32_t* count, int T, const int64_t* pos_dev, int64_t pos0, void* stream) {
    if (!caches || !path || !count) {
        set_error("cache_keep: null pointer argument");
        return SCMX_ERR_ARG;
    }
    if (layers < 0 || layers > 1024 || T < 1 || T > 64) {
        set_error("cache_keep: need up to 1024 layers and 1..64 rows (layers=%d T=%d)", layers, T);
        return SCMX_ERR_ARG;
    }
    if (int rc = check_cache("cache_keep", 1, hk, d, cache_rows, T, pos_dev, pos0)) return rc;
    if (layers == 0) return SCMX_OK;
    const int each = eight ? 4 : 2;
    for (int i = 0; i < layers * each; ++i)
        if (!caches[i] || (i % each < 2 && caches[i] % 16)) {
            set_error("cache_keep: layer %d has a null or misaligned pointer", i / each);
            return SCMX_ERR_ARG;
        }
    uint64_t sorted[4 * 1024];   // the same rows moved twice at once would race
    std::copy(caches, caches + layers * each, sorted);
    std::sort(sorted, sorted + layers * each);
    if (std::adjacent_find(sorted, sorted + layers * each) != sorted + layers * each) {
        set_error("cache_keep: a cache is given twice");
        return SCMX_ERR_ARG;
    }
    for (int l0 = 0; l0 < layers; l0 += KEEP_LAYERS) {
        KeepArgs a{};
        const int n = layers - l0 < KEEP_LAYERS ? layers - l0 : KEEP_LAYERS;
        for (int l = 0; l < n; ++l)
            for (int i = 0; i < each; ++i) a.t[l][i] = reinterpret_cast<void*>(uintptr_t(caches[size_t(l0 + l) * each + i]));
        const auto go = [&](auto rowb) {
            cache_keep_kernel<decltype(rowb)::value>
                <<<dim3(hk, 2, n), dim3(CNT), 0, (hipStream_t)stream>>>(a, eight != 0, cache_rows, path, count, T, pos_dev, pos0);
        };
        switch (eight ? d : 2 * d) {
            case 64: go(std::integral_constant<int, 64>{}); break;
            case 128: go(std::integral_constant<int, 128>{}); break;
            case 256: go(std::integral_constant<int, 256>{}); break;
            default: go(std::integral_constant<int, 512>{}); break;
        }
    }
    return check_launch("cache_keep");
}
