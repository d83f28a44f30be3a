// Rows to MXFP4 and back (include/scmx_mx.h, scmx_mx_quantize and scmx_mx_dequantize).
//
// A lane holds eight consecutive values, four lanes a block of 32: the block's largest magnitude over a quad by two row operations, its
// byte from that exponent, the codes by the FP4 conversions, which round to nearest even and hold what passes 6 to 6.  Bound by memory.
#include <type_traits>

#include "mx.h"

namespace scmx {

constexpr int QNT = 256, QPIECES = 4;   // pieces of 512 values that a wave takes of a row at once

// Blocks in two dimensions: a launch's threads in one are below 2^32.
static dim3 grid_of(uint64_t blocks) {
    const uint64_t x = blocks < (1u << 22) ? blocks : 1u << 22;
    return dim3(unsigned(x), unsigned((blocks + x - 1) / x));
}
__device__ __forceinline__ uint64_t block_index() { return uint64_t(blockIdx.y) * gridDim.x + blockIdx.x; }

template <int TYPE>
struct Raw8 {
    u32x4 w[TYPE == SCMX_MX_F32 ? 2 : 1];
};
template <int TYPE, bool ALIGNED>
__device__ __forceinline__ Raw8<TYPE> load8(const void* x, size_t at) {
    Raw8<TYPE> r;
    if constexpr (ALIGNED) {
        const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const char*>(x) + at * (TYPE == SCMX_MX_F32 ? 4 : 2));
        r.w[0] = p[0];
        if constexpr (TYPE == SCMX_MX_F32) r.w[1] = p[1];
    } else if constexpr (TYPE == SCMX_MX_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.w[i / 4][i % 4] = static_cast<const uint32_t*>(x)[at + i];
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(x) + at;
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[0][i] = p[2 * i] | uint32_t(p[2 * i + 1]) << 16;
    }
    return r;
}
template <int TYPE>
__device__ __forceinline__ void floats(const Raw8<TYPE>& r, float* x) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (TYPE == SCMX_MX_F32) x[i] = __uint_as_float(r.w[i / 4][i % 4]);
        else if constexpr (TYPE == SCMX_MX_BF16) x[i] = i % 2 ? bf16_hi(r.w[0][i / 2]) : bf16_lo(r.w[0][i / 2]);
        else x[i] = float(__builtin_bit_cast(_Float16, uint16_t(r.w[0][i / 2] >> (16 * (i % 2)))));
    }
}

// A wave per 2048 values of a row.
template <int TYPE, bool ALIGNED>
__global__ __launch_bounds__(QNT) void mx_quantize_kernel(const void* __restrict__ x, int64_t ldx, uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales, int M, int K, int chunks) {
    const int lane = threadIdx.x & 63;
    const uint64_t unit = block_index() * (QNT / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), at = unit / uint32_t(chunks);
    if (at >= uint64_t(M)) return;
    const int row = int(at), k0 = int(unit - at * uint32_t(chunks)) * (512 * QPIECES) + 8 * lane;
    Raw8<TYPE> r[QPIECES];
#pragma unroll
    for (int p = 0; p < QPIECES; ++p)   // (behind the row's end: its last values again)
        r[p] = load8<TYPE, ALIGNED>(x, size_t(int64_t(row) * ldx) + min(k0 + 512 * p, K - 8));
#pragma unroll
    for (int p = 0; p < QPIECES; ++p) {
        const int k = k0 + 512 * p;
        float f[8];
        floats<TYPE>(r[p], f);
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7FFFFFFFu);
        const uint32_t byte = mx_byte(quad_max(top)), w = mx_codes(f, byte);
        if (k < K) {   // (a block is whole or absent)
            *reinterpret_cast<uint32_t*>(codes + size_t(row) * (K / 2) + k / 2) = w;
            if (lane % 4 == 0) scales[size_t(row) * (K / 32) + k / 32] = uint8_t(byte);
        }
    }
}

// A sum over a wave's lanes, in each of them: row operations within sixteen lanes, then the four rows.
template <int CTRL>
__device__ __forceinline__ double dpp_add(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return v + __builtin_bit_cast(double, uint64_t(dpp<CTRL>(uint32_t(b >> 32))) << 32 | dpp<CTRL>(uint32_t(b)));
}
__device__ __forceinline__ double wave_sum(double v) {
    v = dpp_add<ROW_MIRROR>(dpp_add<HALF_MIRROR>(dpp_add<QUAD_SWAP2>(dpp_add<QUAD_SWAP1>(v))));
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    double sum = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const uint32_t hi = uint32_t(__builtin_amdgcn_readlane(int(b >> 32), 16 * r));
        const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(b), 16 * r));
        sum += __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
    }
    return sum;
}

// RMSNorm first: WPR waves a row, NC pieces of 8 values a lane.  The codes are those of the float64 values: a product rounded to float32
// lands on the other side of a border between codes once in a million values, a third of the block's largest value off.  The sum of
// squares is in float64.  A value times its gain is exact in float32; times the inverse less and more 2^-21 of it, which is rounded to
// within 3 * 2^-24, float64's result lies between the two, and if both take the same code and byte, so does it.  If not, once in some
// thousand pieces, or where a product leaves float32's range, the wave takes its piece in float64.  In a graph 8192 rows of 2048 take
// 11.4-11.8 us, 32768 33.5-33.9 (without the norm 6.5-7.0, 25.0-25.7: memory); all in float64 16.8, its instructions.
template <int NC, int WPR, bool ALIGNED>
__global__ __launch_bounds__(QNT, NC > 4 ? 2 : 4) void mx_norm_quantize_kernel(const uint16_t* __restrict__ x, int64_t ldx,
                                                                               const uint16_t* __restrict__ nw, float eps,
                                                                               uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                               int M, int K) {
    __shared__ double s_sum[QNT / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = wave % WPR * 64 + lane;
    const uint64_t unit = block_index() * (QNT / 64 / WPR) + wave / WPR;
    if (unit >= uint64_t(M)) return;   // (a row's waves together)
    const int row = int(unit);
    Raw8<SCMX_MX_BF16> r[NC];
    const size_t at = size_t(int64_t(row) * ldx);
#pragma unroll
    for (int c = 0; c < NC; ++c) r[c] = load8<SCMX_MX_BF16, ALIGNED>(x, at + min((c * 64 * WPR + t) * 8, K - 8));
    double ss = 0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        float f[8];
        floats<SCMX_MX_BF16>(r[c], f);
        double part = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) part = __builtin_fma(double(f[i]), double(f[i]), part);
        if ((c * 64 * WPR + t) * 8 < K) ss += part;
    }
    ss = wave_sum(ss);
    if constexpr (WPR > 1) {
        if (lane == 0) s_sum[wave] = ss;
        __syncthreads();
        ss = 0;
#pragma unroll
        for (int w = 0; w < WPR; ++w) ss += s_sum[wave / WPR * WPR + w];
    }
    const double inv = 1.0 / sqrt(ss / double(K) + double(eps));
    const float inv32 = float(inv), less = inv32 * (1.0f - 0x1p-21f), more = inv32 * (1.0f + 0x1p-21f);
    // (not for an infinity or a NaN in the row; a product with a gain that float32 cannot hold, below 2^-126, is then a zero of blocks from
    // 2^-58 on)
    const bool plain = inv32 > 0x1p-120f && inv32 < 0x1p60f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int k = (c * 64 * WPR + t) * 8;
        float f[8], g[8], below[8], above[8];
        floats<SCMX_MX_BF16>(r[c], f);
        floats<SCMX_MX_BF16>(load8<SCMX_MX_BF16, ALIGNED>(nw, min(k, K - 8)), g);
        int32_t plus = INT32_MIN;
        uint32_t minus = 0;   // as bits the largest of either sign, a NaN above all others
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = f[i] * g[i];
            plus = max(plus, int32_t(__float_as_uint(v)));
            minus = max(minus, __float_as_uint(v));
            below[i] = v * less;
            above[i] = v * more;
        }
        const float top = __uint_as_float(quad_max(max(uint32_t(plus) & 0x7FFFFFFFu, minus & 0x7FFFFFFFu)));
        const uint32_t e = __float_as_uint(top * more) >> 23;
        uint32_t byte = e - 2, w = mx_codes_finite(above, byte);
        const bool sure = plain && e - 69u <= 254u - 69u && e == __float_as_uint(top * less) >> 23 && w == mx_codes_finite(below, byte);
        if (__any(!sure)) {
            double d[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = double(f[i]) * inv * double(g[i]);
            w = mx_codes_f64(d, byte);
        }
        if (k < K) {
            *reinterpret_cast<uint32_t*>(codes + size_t(row) * (K / 2) + k / 2) = w;
            if (lane % 4 == 0) scales[size_t(row) * (K / 32) + k / 32] = uint8_t(byte);
        }
    }
}

// Eight values a lane, a word of codes; four lanes share a block's byte.
template <bool F32>
__global__ __launch_bounds__(QNT) void mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                            void* __restrict__ out, uint64_t words) {
    const uint64_t i = block_index() * QNT + threadIdx.x;   // of eight values
    if (i >= words) return;
    const uint32_t w = reinterpret_cast<const uint32_t*>(codes)[i];
    const float s = mx_scale(scales[i / 4]);
    if constexpr (F32) {
        f32x4* o = static_cast<f32x4*>(out) + 2 * i;
        const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1),
                    c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3);
        o[0] = f32x4{a[0], a[1], b[0], b[1]};
        o[1] = f32x4{c[0], c[1], d[0], d[1]};
    } else {
        static_cast<u32x4*>(out)[i] = u32x4{mx_bf16x2<0>(w, s), mx_bf16x2<1>(w, s), mx_bf16x2<2>(w, s), mx_bf16x2<3>(w, s)};
    }
}

template <int NC, bool ALIGNED>
static void launch_norm(const void* x, int64_t ldx, const uint16_t* nw, float eps, uint8_t* codes, uint8_t* scales, int M, int K, int wpr,
                        hipStream_t st) {
    const uint16_t* p = static_cast<const uint16_t*>(x);
    const dim3 fours = grid_of((uint64_t(M) + 3) / 4);
    if (wpr == 1) mx_norm_quantize_kernel<NC, 1, ALIGNED><<<fours, dim3(QNT), 0, st>>>(p, ldx, nw, eps, codes, scales, M, K);
    else mx_norm_quantize_kernel<NC, 4, ALIGNED><<<grid_of(M), dim3(QNT), 0, st>>>(p, ldx, nw, eps, codes, scales, M, K);
}

}  // namespace scmx

using namespace scmx;

extern "C" int scmx_mx_quantize(const void* x, int type, int64_t ldx, const uint16_t* nw, float eps, uint8_t* codes, uint8_t* scales, int M,
                                int K, void* stream) {
    if (M < 0 || K < 32 || K % 32 || K > (1 << 30) || (type != SCMX_MX_BF16 && type != SCMX_MX_F16 && type != SCMX_MX_F32)) {
        set_error("mx_quantize: need rows of a multiple of 32 values, up to 2^30, in bf16, fp16 or float32 (M=%d K=%d type=%d)", M, K,
                  type);
        return SCMX_ERR_ARG;
    }
    if (M && (!x || !codes || !scales)) {
        set_error("mx_quantize: null pointer argument");
        return SCMX_ERR_ARG;
    }
    if (nw && (type != SCMX_MX_BF16 || K > 16384)) {
        set_error("mx_quantize: the norm takes bf16 rows of up to 16384 values (K=%d type=%d)", K, type);
        return SCMX_ERR_ARG;
    }
    if (M > 1 && (ldx < K || ldx > INT64_MAX / 8 / M)) {
        set_error("mx_quantize: rows of %d values are %lld apart", K, (long long)ldx);
        return SCMX_ERR_ARG;
    }
    const int size = type == SCMX_MX_F32 ? 4 : 2;
    if (uintptr_t(x) % size || uintptr_t(nw) % 2 || uintptr_t(codes) % 16) {
        set_error("mx_quantize: codes must be 16-byte aligned, x and nw as their types");
        return SCMX_ERR_ARG;
    }
    if (M == 0) return SCMX_OK;
    if (M == 1) ldx = K;
    const hipStream_t st = (hipStream_t)stream;
    const bool aligned = (uintptr_t(x) | uintptr_t(nw)) % 16 == 0 && (M == 1 || ldx * size % 16 == 0);
    if (nw) {
        // a wave a row where the rows are many and short enough for its registers, else four: 1024 / 2048 / 8192 rows of 2048 3.8 / 4.5 /
        // 11.4 us, with four waves 3.3 / 4.7 / 12.8, 4096 rows of 1024 4.0 and 6.8
        const int wpr = K <= 2048 && M >= 2048 ? 1 : 4, pieces = (K / 8 + 64 * wpr - 1) / (64 * wpr);
        const auto go = [&](auto nc) {
            constexpr int NC = decltype(nc)::value;
            if (aligned) launch_norm<NC, true>(x, ldx, nw, eps, codes, scales, M, K, wpr, st);
            else launch_norm<NC, false>(x, ldx, nw, eps, codes, scales, M, K, wpr, st);
        };
        if (pieces <= 1) go(std::integral_constant<int, 1>{});
        else if (pieces <= 2) go(std::integral_constant<int, 2>{});
        else if (pieces <= 4) go(std::integral_constant<int, 4>{});
        else go(std::integral_constant<int, 8>{});
        return check_launch("mx_quantize");
    }
    const int chunks = (K + 512 * QPIECES - 1) / (512 * QPIECES);
    const uint64_t blocks = (uint64_t(M) * chunks + QNT / 64 - 1) / (QNT / 64);
    if (blocks > (uint64_t(1) << 37)) {
        set_error("mx_quantize: too many values (M=%d K=%d)", M, K);
        return SCMX_ERR_ARG;
    }
    const auto go = [&](auto t) {
        constexpr int TYPE = decltype(t)::value;
        if (aligned) mx_quantize_kernel<TYPE, true><<<grid_of(blocks), dim3(QNT), 0, st>>>(x, ldx, codes, scales, M, K, chunks);
        else mx_quantize_kernel<TYPE, false><<<grid_of(blocks), dim3(QNT), 0, st>>>(x, ldx, codes, scales, M, K, chunks);
    };
    if (type == SCMX_MX_BF16) go(std::integral_constant<int, SCMX_MX_BF16>{});
    else if (type == SCMX_MX_F16) go(std::integral_constant<int, SCMX_MX_F16>{});
    else go(std::integral_constant<int, SCMX_MX_F32>{});
    return check_launch("mx_quantize");
}

extern "C" int scmx_mx_dequantize(const uint8_t* codes, const uint8_t* scales, void* out, int type, int M, int K, void* stream) {
    if (M < 0 || K < 32 || K % 32 || (type != SCMX_MX_BF16 && type != SCMX_MX_F32)) {
        set_error("mx_dequantize: need rows of a multiple of 32 values, to bf16 or float32 (M=%d K=%d type=%d)", M, K, type);
        return SCMX_ERR_ARG;
    }
    if (M && (!codes || !scales || !out)) {
        set_error("mx_dequantize: null pointer argument");
        return SCMX_ERR_ARG;
    }
    if ((uintptr_t(codes) | uintptr_t(out)) % 16) {
        set_error("mx_dequantize: codes and out must be 16-byte aligned");
        return SCMX_ERR_ARG;
    }
    const uint64_t words = uint64_t(M) * (K / 8), blocks = (words + QNT - 1) / QNT;
    if (blocks > (uint64_t(1) << 37)) {
        set_error("mx_dequantize: too many values (M=%d K=%d)", M, K);
        return SCMX_ERR_ARG;
    }
    if (M == 0) return SCMX_OK;
    const hipStream_t st = (hipStream_t)stream;
    if (type == SCMX_MX_F32) mx_dequantize_kernel<true><<<grid_of(blocks), dim3(QNT), 0, st>>>(codes, scales, out, words);
    else mx_dequantize_kernel<false><<<grid_of(blocks), dim3(QNT), 0, st>>>(codes, scales, out, words);
    return check_launch("mx_dequantize");
}
