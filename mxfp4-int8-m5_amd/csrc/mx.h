// Device side of microscaled 4-bit values (include/scmx_mx.h): blocks of 32 that four neighbouring lanes hold, eight values each.
#pragma once
#include "../../include/scmx_mx.h"
#include "scmx_common.h"

namespace scmx {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// The value of lane l of a row of 16 by a row operation.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 0xF, 0xF, true));
}
constexpr int QUAD_SWAP1 = 0xB1, QUAD_SWAP2 = 0x4E, HALF_MIRROR = 0x141, ROW_MIRROR = 0x140, ROW_SHARE = 0x150;

__device__ __forceinline__ uint32_t quad_max(uint32_t v) {   // over four lanes, in each of them
    v = max(v, dpp<QUAD_SWAP1>(v));
    return max(v, dpp<QUAD_SWAP2>(v));
}

// What the conversions take for the E8M0 byte b: they read the exponent field alone (0 is 2^-127, 255 gives NaN).
__device__ __forceinline__ float mx_scale(uint32_t b) { return __uint_as_float(b << 23); }

// The byte of a block whose largest magnitude has these float bits (NaN and infinities are above all others): the exponent less 2.
__device__ __forceinline__ uint32_t mx_byte(uint32_t top) {
    const uint32_t e = top >> 23;
    return e == 255 ? 255 : e < 2 ? 0 : e - 2;
}

// Eight float values of a lane to a word of codes, for the byte of their block.
__device__ __forceinline__ uint32_t mx_codes_finite(const float* x, uint32_t byte) {
    const float s = mx_scale(byte);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
}
__device__ __forceinline__ uint32_t mx_codes(const float* x, uint32_t byte) { return byte == 255 ? 0 : mx_codes_finite(x, byte); }
// The same of eight bf16 values, packed.
__device__ __forceinline__ uint32_t mx_codes_bf16(u32x4 x, uint32_t byte) {
    const float s = mx_scale(byte);
    const uint32_t a = x[0], b = x[1], c = x[2], d = x[3];   // (a bit cast of a vector's element takes the first)
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, a), s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, b), s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, c), s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2, d), s, 3);
    return byte == 255 ? 0 : w;
}

// Values in float64 (a norm's, a rotation's) go through a float rounded to odd (cut off, the last bit set if anything was), so that none
// lands on the border of two codes that was beside it.  Magnitudes are held to 2^-120 .. 2^128 on the way, and the byte to 10 and above,
// below which 2^-120 would count.
__device__ __forceinline__ uint32_t high(double v) { return uint32_t(__builtin_bit_cast(uint64_t, v) >> 32); }
__device__ __forceinline__ float odd_float(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t hi = uint32_t(b >> 32), lo = uint32_t(b);
    const uint32_t m = min(max(hi & 0x7FFFFFFFu, uint32_t(1023 - 120) << 20), 0x47EFFFFFu);
    const uint32_t cut = ((m << 3) | (lo >> 29)) + 0x40000000u;   // the exponent less 896, to float's
    return __uint_as_float((hi & 0x80000000u) | cut | uint32_t((lo & 0x1FFFFFFFu) != 0));
}
// The byte for the largest magnitude's upper word: exponent fields, float64's less 1023, less 2, plus 127; at most 252 (2^125, of which 6
// is below 2^128).
__device__ __forceinline__ uint32_t mx_byte_f64(uint32_t top) {
    return top >= 0x7FF00000u ? 255 : min(max(top >> 20, 898u + 10u) - 898u, 252u);
}
// Eight values of a lane, of a block that four lanes hold, to a word of codes; byte: the block's.
__device__ __forceinline__ uint32_t mx_codes_f64(const double* v, uint32_t& byte) {
    uint32_t top = 0;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        top = max(top, high(v[i]) & 0x7FFFFFFFu);
        x[i] = odd_float(v[i]);
    }
    byte = mx_byte_f64(quad_max(top));
    return mx_codes(x, byte);
}
// Byte B of a word of codes as two bf16 values in a word.
template <int B>
__device__ __forceinline__ uint32_t mx_bf16x2(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, B));
}

}  // namespace scmx
