/* scmx, microscaled 4-bit values (MXFP4): entry points of libscmx.so beside those of scmx.h and scmx_cache.h, under the same rules
 * (device pointers, the caller's stream, no allocation, no synchronisation, no state, SCMX_ERR_* and scmx_last_error()).
 * The reference has none of these: its activations are INT8 and its cache holds the model's type.
 *
 * A tensor of rows of K values, K a multiple of 32, is a pair: codes uint8 [rows, K / 2], two E2M1 codes a byte, the even value in the low
 * four bits (sign, then an index into 0, 0.5, 1, 1.5, 2, 3, 4, 6), and scales uint8 [rows, K / 32], an E8M0 byte for each 32 values:
 * value = E2M1 * 2^(byte - 127), byte 255: all 32 are NaN.  4.25 bits a value; what a standard MXFP4 checkpoint holds.
 * Values become codes by one rule everywhere: byte - 127 = floor(log2 of the block's largest magnitude) - 2, at least -127, each value
 * over 2^(byte - 127) rounded to the nearest E2M1, ties to the even code, what passes 6 held to 6; a block with a NaN or an infinity
 * takes the byte 255 (codes 0).
 * codes are 16-byte aligned, scales at any address. */
#ifndef SCMX_MX_H
#define SCMX_MX_H

#include "scmx.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SCMX_MX_BF16 0
#define SCMX_MX_F16 1
#define SCMX_MX_F32 2

/* x [M, K] of `type` (K <= 2^30), row i at element i * ldx (ldx >= K, any alignment), to codes and scales.  With nw (bf16 [K]; x bf16,
 * K <= 16384): of the rows' RMSNorm x / sqrt(mean(x^2) + eps) * nw, in float64, so that a value beside the border of two codes takes its
 * own; there byte is at least 10, and magnitudes from 2^128 on count as the largest below. */
int scmx_mx_quantize(const void* x, int type, int64_t ldx, const uint16_t* nw, float eps, uint8_t* codes, uint8_t* scales, int M,
                     int K, void* stream);

/* The values of M rows of K as bf16 or float32 (type; 16-byte aligned): exact but where they pass that type's range. */
int scmx_mx_dequantize(const uint8_t* codes, const uint8_t* scales, void* out, int type, int M, int K, void* stream);

/* x w^T of MXFP4 operands, x of M rows and w of N rows of K values, on the scaled matrix instructions, sums in float32, each result rounded
 * once to bf16.  epi 1: out [M, N]; 2: + res [M, N]; 3: silu(gate) * up of w rows in the order of the SwiGLU epilogue of scmx.h (two gates,
 * their two ups; N a multiple of 4), out [M, N / 2].
 * K <= 2^23; M and N below 2^31 - 511 (any M where N times K is below 512); N <= 2^26 where M <= 16 or M times K is below 512; fewer than
 * 2^31 groups of 16 x 16 results.  What is beyond is refused. */
int scmx_mx_mm(const uint8_t* xcodes, const uint8_t* xscales, const uint8_t* wcodes, const uint8_t* wscales, const uint16_t* res,
               uint16_t* out, int epi, int M, int N, int K, void* stream);

/* scmx_mx_quantize (bf16, with nw or without) and scmx_mx_mm in one call.  workspace: scmx_mx_linear_workspace(M, N, K, nw != NULL) bytes
 * (0: none), 16-byte aligned; it holds the rows' codes and scales between the call's launches. */
size_t scmx_mx_linear_workspace(int M, int N, int K, int norm);
int scmx_mx_linear(const uint16_t* x, int64_t ldx, const uint16_t* nw, float eps, const uint8_t* wcodes, const uint8_t* wscales,
                   const uint16_t* res, uint16_t* out, int epi, int M, int N, int K, void* workspace, size_t workspace_bytes,
                   void* stream);

/* ---- a KV cache of such rows: codes uint8 [hk, cache_rows, d / 2] and scales uint8 [hk, cache_rows, d / 32], for K and for V.  What
 * scmx_cache.h says of positions, trees and head dims (64, 128, 256) holds here; scales are aligned to d / 32 bytes. ---- */

/* scmx_cache_write into such a cache.  Norm, rotation and codes in float64 (the RMSNorm's rule above for keys; values are coded as they
 * are): a row next to the border of two codes takes the definition's. */
int scmx_cache4_write(const int32_t* acc, const float* xscale, const float* wscale, const uint16_t* y, const uint16_t* qn,
                      const uint16_t* kn, float eps, uint16_t* q, uint8_t* kcache, uint8_t* vcache, uint8_t* kscale, uint8_t* vscale,
                      int L, int hq, int hk, int d, const float* inv_freq, const int32_t* depth, const int64_t* pos_dev,
                      int64_t pos0, int cache_rows, void* stream);

/* Rows row0 .. row0 + n - 1 as bf16: k, v [hk, n, d]. */
int scmx_cache4_read(const uint8_t* kcache, const uint8_t* vcache, const uint8_t* kscale, const uint8_t* vscale, uint16_t* k, uint16_t* v,
                     int hk, int d, int cache_rows, int row0, int n, void* stream);

/* scmx_cache_keep; caches: HOST array of layers * 4 device pointers, a layer's K, V and their scales. */
int scmx_cache4_keep(const uint64_t* caches, int layers, int hk, int d, int cache_rows, const int32_t* path, const int32_t* count, int T,
                     const int64_t* pos_dev, int64_t pos0, void* stream);

/* scmx_attn_tree over such a cache.  q . K^T is taken to float32: q as two E4M3 parts a block of 32, whose sum differs from q by at most
 * 2^-23 of the block's largest value, times K as it is held.  The probabilities are held in 16 bits, as two bf16 parts, in the sum and in
 * the denominator alike (2^-15 of sum p |v| at most).  Values of any size: sums of 6 * 2^125 over 2^31 rows stay in float32; where a query
 * meets p |v| from 2^90 on, probabilities below 2^-80 of its largest may count as none.  A row's NaN reaches the nodes that see it and no
 * other.  Scale bytes of rows that are read are at most 252, as the append's are, or 255. */
int scmx_attn_tree4_splits(int T, int n, int hq, int hk, int d);
int scmx_attn_tree4(const uint16_t* q, const uint8_t* kcache, const uint8_t* vcache, const uint8_t* kscale, const uint8_t* vscale,
                    const int64_t* mask, const int64_t* pos_dev, int64_t pos0, uint16_t* out, int T, int hq, int hk, int d,
                    int cache_rows, float scale, float* workspace, int splits, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SCMX_MX_H */
