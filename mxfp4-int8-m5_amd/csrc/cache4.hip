// A KV cache in 4 bits (include/scmx_mx.h): the append of new tokens (norm, rotary embedding, codes in one pass), the read-back for a
// prompt's attention, and the accepted rows of a tree of drafts moved together.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "mx.h"

namespace scmx {

constexpr int CNT = 256;
constexpr unsigned WIDE = 1u << 22;   // workgroups of a launch in x at most (its threads in one dimension are below 2^32), the others in z
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(4)));

struct Write4Args {
    const int32_t* acc;
    const float* xscale;
    const float* wscale;
    const uint16_t* y;
    const uint16_t* qn;
    const uint16_t* kn;
    float eps;
    uint16_t* q;
    uint8_t* cache[2];   // K, V
    uint8_t* scale[2];
    int L, hq, hk;
    const float* inv_freq;
    const int32_t* depth;
    const int64_t* pos_dev;
    int64_t pos0;
    int rows;
};

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, uint64_t(dpp<CTRL>(uint32_t(b >> 32))) << 32 | dpp<CTRL>(uint32_t(b)));
}
// The sum over the LPH lanes of a head (8, 16 or 32, aligned), in every lane.
template <int LPH>
__device__ __forceinline__ double head_sum(double v) {
    v += dpp64<QUAD_SWAP1>(v);
    v += dpp64<QUAD_SWAP2>(v);
    v += dpp64<HALF_MIRROR>(v);
    if (LPH >= 16) v += dpp64<ROW_MIRROR>(v);
    if (LPH >= 32) v += __shfl_xor(v, 16, WAVE);
    return v;
}
template <int LPH>
__device__ __forceinline__ double half_away(double v) {   // of the lane half a head away
    if (LPH == 8) return dpp64<0x1B>(dpp64<HALF_MIRROR>(v));          // 7 - j, then its quad reversed: j ^ 4
    if (LPH == 16) return dpp64<0x128>(v);                            // row_ror 8
    return __shfl_xor(v, 16, WAVE);
}

// Whether f lies in the middle of two bf16 numbers: only there does a float64's rounding to float decide the next one's.
__device__ __forceinline__ bool tie(float f) { return (__float_as_uint(f) & 0xFFFFu) == 0x8000u; }
// f, the float of v, and where that is such a middle and v is not its neighbour on v's side.
__device__ __forceinline__ float beside(float f, double v) {
    const double back = f;
    const uint32_t b = __float_as_uint(f);
    return !tie(f) || back == v ? f : __uint_as_float(fabs(back) > fabs(v) ? b - 1 : b + 1);
}

// One token per blockIdx.x (and z, from WIDE tokens on).  A head of D values is held by D / 8 lanes, eight consecutive values each; four
// lanes hold a block of 32.  Per head (x: the row, n: its norm)
//     n = x / sqrt(mean(x^2) + eps) * w,  (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * inv_freq
// in float64 throughout: a float32 rounding before a code's lands on the other side of a border once in a million values, and a third of
// the block's largest value off (before a query's to bf16: once in a hundred thousand, by its last bit).  The angle in turns is off by
// 2^-53 of their number.
template <int D, bool ACC>
__global__ __launch_bounds__(CNT) void cache4_write_kernel(const Write4Args a) {
    constexpr int LPH = D / 8, GROUPS = CNT / LPH;
    __shared__ double s_sin[D / 2], s_cos[D / 2];
    const unsigned token = blockIdx.z * gridDim.x + blockIdx.x;
    if (token >= unsigned(a.L)) return;
    const int row = int(token), grp = threadIdx.x / LPH, j = threadIdx.x % LPH;
    const int heads = a.hq + 2 * a.hk, stride = gridDim.y * GROUPS;
    const int64_t pos = a.pos_dev ? a.pos_dev[0] : a.pos0;
    const bool fits = pos >= 0 && pos <= int64_t(a.rows) - a.L;
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
        sincospi(2.0 * (turns - rint(turns)), &s_sin[threadIdx.x], &s_cos[threadIdx.x]);
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
        const int h = g - a.hq - (is_v ? a.hk : 0);
        uint32_t codes, byte;
        if (is_v) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
            byte = mx_byte(quad_max(top));
            codes = mx_codes(x, byte);
        } else {
            double v[8], ss = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __builtin_fma(double(x[i]), double(x[i]), ss);
            ss = head_sum<LPH>(ss);
            const double inv = 1.0 / sqrt(ss / double(D) + double(a.eps));
            const u32x4 w = g < a.hq ? wq : wk;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = double(x[i]) * inv * double(i % 2 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]));
            const int at = 8 * (j % (LPH / 2));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const double other = half_away<LPH>(v[i]) * s_sin[at + i];
                v[i] = __builtin_fma(v[i], s_cos[at + i], j < LPH / 2 ? -other : other);
            }
            if (g < a.hq) {
                u32x4 o;
                float f[8];
                bool ties = false;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    f[i] = float(v[i]);
                    ties |= tie(f[i]);
                }
                if (ties) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = beside(f[i], v[i]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = f32_to_bf16x2(f[2 * i], f[2 * i + 1]);
                *reinterpret_cast<u32x4*>(a.q + (size_t(row) * a.hq + g) * D + 8 * j) = o;
                continue;
            }
            codes = mx_codes_f64(v, byte);
        }
        if (!fits) continue;
        const size_t at = size_t(h) * a.rows + size_t(pos) + row;
        *reinterpret_cast<uint32_t*>(a.cache[is_v] + at * (D / 2) + 4 * j) = codes;
        if (j % 4 == 0) a.scale[is_v][at * (D / 32) + j / 4] = uint8_t(byte);
    }
}

// Eight values a lane, a word of codes; blockIdx.y: KV head, blockIdx.z % 2: K or V.
__global__ __launch_bounds__(CNT) void cache4_read_kernel(const uint8_t* kc, const uint8_t* vc, const uint8_t* ks, const uint8_t* vs,
                                                          uint16_t* k, uint16_t* v, int d, int rows, int row0, int n) {
    const size_t first = size_t(blockIdx.y) * rows + row0;
    const bool is_v = blockIdx.z % 2;
    const uint8_t* codes = (is_v ? vc : kc) + first * (d / 2);
    const uint8_t* scales = (is_v ? vs : ks) + first * (d / 32);
    uint16_t* out = (is_v ? v : k) + size_t(blockIdx.y) * n * d;
    const size_t i = (size_t(blockIdx.z / 2) * gridDim.x + blockIdx.x) * CNT + threadIdx.x;   // of eight values
    if (i >= size_t(n) * (d / 8)) return;
    const uint32_t w = reinterpret_cast<const uint32_t*>(codes)[i];
    const float s = mx_scale(scales[i / 4]);
    reinterpret_cast<u32x4*>(out)[i] = u32x4{mx_bf16x2<0>(w, s), mx_bf16x2<1>(w, s), mx_bf16x2<2>(w, s), mx_bf16x2<3>(w, s)};
}

// The layers of one launch: their pointers travel in the kernel's arguments.
constexpr int KEEP_LAYERS = 32;
struct Keep4Args {
    uint8_t* t[KEEP_LAYERS][4];
};

// blockIdx.x: KV head, y: K or V, z: layer.  The rows are read whole before any is written (a row may be both).
template <int D>
__global__ __launch_bounds__(CNT) void cache4_keep_kernel(const Keep4Args a, int rows, const int32_t* path, const int32_t* count, int T,
                                                          const int64_t* pos_dev, int64_t pos0) {
    constexpr int ROWB = D / 2, PER = ROWB / 16, N = (64 * PER + CNT - 1) / CNT;   // 16-byte pieces a row, and a thread
    using Scales = std::conditional_t<D == 64, uint16_t, std::conditional_t<D == 128, uint32_t, uint64_t>>;   // a row's
    const int64_t pos = pos_dev ? pos_dev[0] : pos0;
    if (pos < 0 || pos > int64_t(rows) - T) return;
    const int kept = min(max(count[0], 0), T);
    const size_t first = size_t(blockIdx.x) * rows + size_t(pos);
    uint8_t* t = a.t[blockIdx.z][blockIdx.y] + first * ROWB;
    Scales* s = reinterpret_cast<Scales*>(a.t[blockIdx.z][2 + blockIdx.y]) + first;
    u32x4 w[N];
    int from[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = threadIdx.x + CNT * i, to = c / PER;
        from[i] = to < kept ? path[to] : -1;
        if (from[i] < 0 || from[i] >= T || from[i] == to) from[i] = -1;
        if (from[i] >= 0) w[i] = *reinterpret_cast<const u32x4*>(t + size_t(from[i]) * ROWB + c % PER * 16);
    }
    const int mine = int(threadIdx.x) < kept ? path[threadIdx.x] : -1;
    const bool moves = mine >= 0 && mine < T;
    Scales scale = 0;
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
static int check_cache4(const char* who, int hq, int hk, int d, int rows, int64_t n, const int64_t* pos_dev, int64_t pos0) {
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

extern "C" int scmx_cache4_write(const int32_t* acc, const float* xscale, const float* wscale, const uint16_t* y, const uint16_t* qn,
                                 const uint16_t* kn, float eps, uint16_t* q, uint8_t* kcache, uint8_t* vcache, uint8_t* kscale,
                                 uint8_t* vscale, int L, int hq, int hk, int d, const float* inv_freq, const int32_t* depth,
                                 const int64_t* pos_dev, int64_t pos0, int cache_rows, void* stream) {
    if ((L && ((!acc && !y) || !q)) || (acc && (!xscale || !wscale)) || !qn || !kn || !kcache || !vcache || !inv_freq || !kscale ||
        !vscale) {
        set_error("cache4_write: null pointer argument");
        return SCMX_ERR_ARG;
    }
    if (int rc = check_cache4("cache4_write", hq, hk, d, cache_rows, L, pos_dev, pos0)) return rc;
    if ((uintptr_t(acc ? nullptr : y) | uintptr_t(qn) | uintptr_t(kn) | uintptr_t(q) | uintptr_t(kcache) | uintptr_t(vcache)) % 16 ||
        (uintptr_t(kscale) | uintptr_t(vscale)) % (d / 32)) {
        set_error("cache4_write: y, qn, kn, q and the caches must be 16-byte aligned, scales to a row's bytes");
        return SCMX_ERR_ARG;
    }
    if (kcache == vcache || kscale == vscale) {
        set_error("cache4_write: K and V are one cache");
        return SCMX_ERR_ARG;
    }
    if (L == 0) return SCMX_OK;
    const Write4Args a{acc, xscale,   wscale, y,     qn,      kn,   eps,       q, {kcache, vcache}, {kscale, vscale}, L, hq,
                       hk,  inv_freq, depth,  pos_dev, pos0, cache_rows};
    const int groups = CNT / (d / 8), turns = (hq + 2 * hk + groups - 1) / groups;
    // a few tokens are spread over the CUs; a prompt fills them with a workgroup a token, which then takes the angles once
    const unsigned x = std::min(unsigned(L), WIDE);
    const dim3 grid(x, L >= 256 ? 1 : turns, (unsigned(L) + x - 1) / x);
    const hipStream_t st = (hipStream_t)stream;
    const auto go = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        if (acc) cache4_write_kernel<D, true><<<grid, dim3(CNT), 0, st>>>(a);
        else cache4_write_kernel<D, false><<<grid, dim3(CNT), 0, st>>>(a);
    };
    if (d == 64) go(std::integral_constant<int, 64>{});
    else if (d == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
    return check_launch("cache4_write");
}

extern "C" int scmx_cache4_read(const uint8_t* kcache, const uint8_t* vcache, const uint8_t* kscale, const uint8_t* vscale, uint16_t* k,
                                uint16_t* v, int hk, int d, int cache_rows, int row0, int n, void* stream) {
    if (!kcache || !vcache || !kscale || !vscale || (n && (!k || !v))) {
        set_error("cache4_read: null pointer argument");
        return SCMX_ERR_ARG;
    }
    if (int rc = check_cache4("cache4_read", 1, hk, d, cache_rows, n, nullptr, row0)) return rc;
    if ((uintptr_t(kcache) | uintptr_t(vcache) | uintptr_t(k) | uintptr_t(v)) % 16) {
        set_error("cache4_read: the caches and outputs must be 16-byte aligned");
        return SCMX_ERR_ARG;
    }
    if (n == 0) return SCMX_OK;
    const unsigned blocks = unsigned((size_t(n) * (d / 8) + CNT - 1) / CNT), x = std::min(blocks, WIDE);
    const dim3 grid(x, hk, 2 * ((blocks + x - 1) / x));
    cache4_read_kernel<<<grid, dim3(CNT), 0, (hipStream_t)stream>>>(kcache, vcache, kscale, vscale, k, v, d, cache_rows, row0, n);
    return check_launch("cache4_read");
}

extern "C" int scmx_cache4_keep(const uint64_t* caches, int layers, int hk, int d, int cache_rows, const int32_t* path,
                                const int32_t* count, int T, const int64_t* pos_dev, int64_t pos0, void* stream) {
    if (!caches || !path || !count) {
        set_error("cache4_keep: null pointer argument");
        return SCMX_ERR_ARG;
    }
    if (layers < 0 || layers > 1024 || T < 1 || T > 64) {
        set_error("cache4_keep: need up to 1024 layers and 1..64 rows (layers=%d T=%d)", layers, T);
        return SCMX_ERR_ARG;
    }
    if (int rc = check_cache4("cache4_keep", 1, hk, d, cache_rows, T, pos_dev, pos0)) return rc;
    if (layers == 0) return SCMX_OK;
    for (int i = 0; i < layers * 4; ++i)
        if (!caches[i] || caches[i] % (i % 4 < 2 ? 16 : uint64_t(d / 32))) {
            set_error("cache4_keep: layer %d has a null or misaligned pointer", i / 4);
            return SCMX_ERR_ARG;
        }
    uint64_t sorted[4 * 1024];   // the same rows moved twice at once would race
    std::copy(caches, caches + layers * 4, sorted);
    std::sort(sorted, sorted + layers * 4);
    if (std::adjacent_find(sorted, sorted + layers * 4) != sorted + layers * 4) {
        set_error("cache4_keep: a cache is given twice");
        return SCMX_ERR_ARG;
    }
    for (int l0 = 0; l0 < layers; l0 += KEEP_LAYERS) {
        Keep4Args a{};
        const int n = layers - l0 < KEEP_LAYERS ? layers - l0 : KEEP_LAYERS;
        for (int l = 0; l < n; ++l)
            for (int i = 0; i < 4; ++i) a.t[l][i] = reinterpret_cast<uint8_t*>(uintptr_t(caches[size_t(l0 + l) * 4 + i]));
        const auto go = [&](auto dim) {
            cache4_keep_kernel<decltype(dim)::value>
                <<<dim3(hk, 2, n), dim3(CNT), 0, (hipStream_t)stream>>>(a, cache_rows, path, count, T, pos_dev, pos0);
        };
        if (d == 64) go(std::integral_constant<int, 64>{});
        else if (d == 128) go(std::integral_constant<int, 128>{});
        else go(std::integral_constant<int, 256>{});
    }
    return check_launch("cache4_keep");
}
