/* scmx, drafted tokens over a (quantised) KV cache: entry points of libscmx.so beside those of scmx.h, under the same rules
 * (device pointers, the caller's stream, no allocation, no synchronisation, no state, SCMX_ERR_* and scmx_last_error()).
 * The reference has none of these: its decode step takes one token, its cache holds the model's type.
 *
 * A cache is a K and a V tensor (two, not one twice) [hk, cache_rows, d], either bf16 (kscale = vscale = NULL) or INT8 with one
 * float scale per row (kscale, vscale [hk, cache_rows]): value = code * scale.  8-bit rows take d + 4 bytes where bf16 rows take 2 d.
 * A tree of drafted tokens has its T (1..64) nodes in rows pos .. pos + T - 1 behind the pos rows of the sequence, every node
 * after its parent, node 0 the sequence's newest token.  pos is *pos_dev when pos_dev != NULL (a device-resident position, so that a
 * captured graph can be replayed for every step), else pos0.  d is 64, 128 or 256.  Tensors are 16-byte aligned (scales, masks and
 * numbers: as their type).  */
#ifndef SCMX_CACHE_H
#define SCMX_CACHE_H

#include "scmx.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Per-head RMSNorm of q and k (weights qn, kn [d]), rotary embedding (inv_freq [d/2], element e with e + d/2) at position
 * pos + depth[i] (depth NULL: pos + i) and the append of k and v to rows pos .. pos + L - 1 of the caches, in bf16 or 8 bits.
 * Input: y bf16 [>= L, (hq + 2 hk) d], or acc int32 of the same shape with xscale [>= L] and wscale [(hq + 2 hk) d] (then y is
 * bf16(acc * xscale * wscale)).  q: bf16 [L, hq, d].  Computed in float32 (angles in float64), each result rounded once:
 * scmx_qkv_headnorm_rope, which restates the reference's array ops, rounds three times.  8 bits: scale = max|v| / 127 of the row,
 * code = rint(v / scale); a row whose largest value is below 2^-100 is held as zeros, one with a value that is not finite has
 * the scale NaN.  With pos_dev, a position whose rows do not fit the cache appends nothing (q is written). */
int scmx_cache_write(const int32_t* acc, const float* xscale, const float* wscale, const uint16_t* y, const uint16_t* qn,
                     const uint16_t* kn, float eps, uint16_t* q, void* kcache, void* vcache, float* kscale, float* vscale, int L,
                     int hq, int hk, int d, const float* inv_freq, const int32_t* depth, const int64_t* pos_dev, int64_t pos0,
                     int cache_rows, void* stream);

/* Rows row0 .. row0 + n - 1 of an 8-bit cache as bf16: k, v [hk, n, d]. */
int scmx_cache_read(const int8_t* kcache, const int8_t* vcache, const float* kscale, const float* vscale, uint16_t* k, uint16_t* v,
                    int hk, int d, int cache_rows, int row0, int n, void* stream);

/* Row pos + j takes what row pos + path[j] held before the call, for j < *count, in every one of `layers` caches: the accepted
 * line of a tree moved together.  path int32 [T], any order, repeats allowed; an entry outside 0 .. T - 1 leaves its row, *count
 * is held to 0 .. T.  caches: HOST array of layers * (2 or 4) device pointers, a layer's K, V (and with eight != 0 their scales),
 * read before the call returns; no pointer twice.  layers <= 1024.  With pos_dev, a position whose rows do not fit moves nothing. */
int scmx_cache_keep(const uint64_t* caches, int layers, int eight, int hk, int d, int cache_rows, const int32_t* path,
                    const int32_t* count, int T, const int64_t* pos_dev, int64_t pos0, void* stream);

/* Attention of the T nodes of a tree: out bf16 [T, hq * d] = softmax(q . K^T * scale) V, q bf16 [T, hq, d], hq / hk up to 4096.
 * Every node sees the rows below pos; row pos + j is seen by node i if bit j of mask[i] is set (mask NULL: j <= i, a chain).  A node
 * that sees nothing gets zeros; what a node does not see does not reach its result, infinities and NaN among it.  T = 1 is the decode
 * step's attention over an 8-bit cache.  With pos_dev, a position whose rows do not fit the cache gives zeros.
 * Over an 8-bit cache a row weighs by the product of its probability and its V row's scale, a half-precision number of which the
 * largest is 2^8 .. 2^14: products below 2^-22 of the largest lose bits, below 2^-39 they may vanish from the sum.  The denominator
 * is summed from the same products, in float32, over the scales: a row whose product is below 2^-110 of another's may count as not
 * seen.  V scales are 2^-110 .. 2^122, as the append's are, or 0 for a row of zeros, which takes part as one with the scale 2^-80 would
 * (others are not looked for: a negative or subnormal one gives NaN).  Over a bf16 cache the probabilities are rounded to bf16, in the
 * sum and in the denominator alike (2^-8 of sum p |v| at most), and the sum, in float32, is up to 2^8 (pos + T) times the largest
 * |v|: values up to 1e30 over a million rows.  scale is finite, times log2 e too.
 * splits (1..64): ranges the rows are cut into, a workgroup per range, KV head and 16 or 32 query rows; more than one needs
 * `workspace`, float [splits * T * hq * (d + 2)], 16-byte aligned, used between the call's two launches.
 * scmx_attn_tree_splits: how many to take for n rows in all (the cache's, where the position is on the device); 1 for arguments that
 * scmx_attn_tree refuses. */
int scmx_attn_tree_splits(int T, int n, int hq, int hk, int d);
int scmx_attn_tree(const uint16_t* q, const void* kcache, const void* vcache, const float* kscale, const float* vscale,
                   const int64_t* mask, const int64_t* pos_dev, int64_t pos0, uint16_t* out, int T, int hq, int hk, int d,
                   int cache_rows, float scale, float* workspace, int splits, void* stream);

/* Which drafted tokens the target accepts, and the token after them.  tokens int64 [T], parents int32 [T] (parents[i] < i; node 0
 * is the root), logits [T, V] (float32 if logits_f32, else bf16): the target's after each node; NaN counts as -inf.
 * temperature 0: from the root down, a node's first child that holds the lowest-numbered largest logit; *next is that of the
 * last node.  temperature > 0: p = softmax(logits / temperature) in float64; the children of the current node are tried in index
 * order against r, at first p: child c is taken if uniforms[c] * q(x_c) < r(x_c), else r becomes max(r - q, 0), normalised
 * (unless nothing of it is left); when none is taken, *next is the lowest token at which the running sum of r exceeds
 * uniforms[0] times its total.  q is the row of `draft` (float32 [T, V], the distribution that the node's children were drawn
 * from), or with draft == NULL all mass on x_c (a draft's likeliest tokens, tokens from the text).  Either way *next and the
 * accepted tokens are distributed as the target's own.  With a draft at most `siblings` (1..16) children of a node are tried.
 * uniforms float32 [T] in [0, 1): entry 0 for *next, entry c for node c; not read at temperature 0.  A token outside 0 .. V - 1 is
 * never taken.  Out: path int32 [T] (the accepted nodes from node 0 on, then -1), count int32 [1] (at least 1), next int64 [1].
 * V <= 4194304.  workspace: scmx_verify_workspace(...) bytes, 8-byte aligned, used between the call's launches. */
size_t scmx_verify_workspace(int T, int V, int siblings);
int scmx_verify_drafts(const int64_t* tokens, const int32_t* parents, const void* logits, int logits_f32, const float* draft,
                       double temperature, const float* uniforms, int32_t* path, int32_t* count, int64_t* next, int T, int V,
                       int siblings, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SCMX_CACHE_H */
