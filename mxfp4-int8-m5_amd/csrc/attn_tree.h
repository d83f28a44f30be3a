// What the attention of a tree of drafted tokens shares between caches in bf16 or 8 bits (attn_tree.hip) and in 4 bits (attn_tree4.hip): the
// arguments, the ranges of keys, and the kernels that join the ranges' sums.
#pragma once
#include "scmx_common.h"

namespace scmx {

constexpr int TKEYS = 32, TXCDS = 8, JNT = 256;
// Waves of a workgroup.  Four, two workgroups a CU, whose starts and ends overlap, against eight of one (both launches, in a graph): 16
// tokens, 3000 rows of 16:8 x 128, bf16 12.4 -> 10.9 us, one token, 1000 rows, 8 bits 8.8 -> 7.6, 40000 rows 21.2 -> 20.7.
constexpr int TWAVES = 4, TNT = 64 * TWAVES;
// Tiles up to which one range takes all (four a wave): a second launch costs a microsecond more than the steps it saves.
constexpr int TONE = 16;

struct TreeArgs {
    const uint16_t* q;
    const uint8_t* k;
    const uint8_t* v;
    const float* ks;
    const float* vs;
    const int64_t* mask;
    const int64_t* pos_dev;
    int64_t pos0;
    uint16_t* out;
    float* part;      // [T hq][splits][d] sums, then [T hq][splits][2]: reference, denominator
    int T, hq, hk, rows, splits, blocks;   // blocks: of query rows
    uint32_t by_group;                     // 2^32 / (hq / hk), rounded up: r / group as a high product, exact for r group < 2^32
    float scale;      // times log2 e
};

static __device__ __host__ inline int tiles_of(int n) { return n / TKEYS + (n % TKEYS != 0); }   // (n up to 2^31 - 1)
// Tiles of a range, of a context of n keys in all; at least a tile a wave.
static __device__ __host__ inline int range_tiles(int n, int splits) {
    const int tiles = tiles_of(n), even = (tiles + splits - 1) / splits;
    return tiles <= TONE ? TONE : even > TWAVES ? even : TWAVES;
}

// Joins the ranges of one row of [T, hq], a workgroup: D / 4 lanes a range, the ranges dealt to the rest.  Bound by one trip to memory:
// all that a thread reads is requested at once.  RANGES: at most.
template <int D, int RANGES>
static __global__ __launch_bounds__(JNT) void attn_tree_join_kernel(const float* __restrict__ part, uint16_t* __restrict__ out, int T, int hq,
                                                             int rows, int splits, const int64_t* pos_dev, int64_t pos0) {
    constexpr int PARTS = JNT / (D / 4), PER = (RANGES + PARTS - 1) / PARTS;
    __shared__ float s_num[PARTS][D];
    const int lane = threadIdx.x & 63, p = threadIdx.x / (D / 4), e = threadIdx.x % (D / 4) * 4;
    const float* num0 = part + size_t(blockIdx.x) * splits * D + e;
    const float2 ml =
        reinterpret_cast<const float2*>(part + size_t(T) * hq * splits * D)[size_t(blockIdx.x) * splits + min(lane, splits - 1)];
    f32x4 v[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) v[u] = *reinterpret_cast<const f32x4*>(num0 + size_t(min(p + u * PARTS, splits - 1)) * D);
    const int64_t pos = pos_dev ? pos_dev[0] : pos0;
    if (pos < 0 || pos > int64_t(rows) - T) return;   // zeros, written
    const int n = int(pos) + T, per = range_tiles(n, splits), tiles = tiles_of(n), ranges = (tiles + per - 1) / per;
    if (ranges == 1) return;
    const bool mine = lane < ranges && ml.y != 0.0f;   // (0: a range of which the query sees nothing)
    const float mx = wave_max(mine ? ml.x : -__builtin_inff()), w = mine ? __builtin_amdgcn_exp2f(ml.x - mx) : 0.0f;
    const float den = wave_sum(mine ? w * ml.y : 0.0f);
    f32x4 num = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const float f = __shfl(w, min(p + u * PARTS, 63), WAVE);
        const float there = __shfl(mine ? 1.0f : 0.0f, min(p + u * PARTS, 63), WAVE);
        if (there != 0.0f && p + u * PARTS < 64) {
#pragma unroll
            for (int i = 0; i < 4; ++i) num[i] = __builtin_fmaf(f, v[u][i], num[i]);
        }
    }
    *reinterpret_cast<f32x4*>(&s_num[p][e]) = num;
    __syncthreads();
    if (int(threadIdx.x) >= D / 2) return;
    float lo = 0.0f, hi = 0.0f;
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
        lo += s_num[q][2 * threadIdx.x];
        hi += s_num[q][2 * threadIdx.x + 1];
    }
    const float inv = den == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(den);
    *reinterpret_cast<uint32_t*>(out + size_t(blockIdx.x) * D + 2 * threadIdx.x) = f32_to_bf16x2(lo * inv, hi * inv);
}

// The same for up to 8 ranges and a wave a row, four rows a workgroup: the parts of a row meet across lanes.  64 tokens of 32 heads, four
// ranges of 6000 rows 22.9 -> 21.0 us with the attention; with 16 ranges a wave has too much in a row (one token, 4000 rows 8.5 -> 9.0).
template <int D>
static __global__ __launch_bounds__(JNT) void attn_tree_join_rows_kernel(const float* __restrict__ part, uint16_t* __restrict__ out, int T, int hq,
                                                                  int rows, int splits, const int64_t* pos_dev, int64_t pos0) {
    constexpr int LANES = D / 4, PARTS = 64 / LANES, PER = 8 / PARTS;
    const int lane = threadIdx.x & 63, p = lane / LANES, e = lane % LANES * 4;
    const unsigned all = unsigned(T) * hq, row = min(blockIdx.x * (JNT / 64) + threadIdx.x / 64, all - 1);   // (the last one again)
    const float* num0 = part + size_t(row) * splits * D + e;
    const float2 ml = reinterpret_cast<const float2*>(part + size_t(all) * splits * D)[size_t(row) * splits + min(lane % 8, splits - 1)];
    f32x4 v[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u)
        if (u == 0 || u * PARTS < splits) v[u] = *reinterpret_cast<const f32x4*>(num0 + size_t(min(p + u * PARTS, splits - 1)) * D);
    const int64_t pos = pos_dev ? pos_dev[0] : pos0;
    if (pos < 0 || pos > int64_t(rows) - T) return;   // zeros, written
    const int n = int(pos) + T, per = range_tiles(n, splits), tiles = tiles_of(n), ranges = (tiles + per - 1) / per;
    if (ranges == 1) return;
    const bool mine = lane % 8 < ranges && ml.y != 0.0f;   // (0: a range of which the query sees nothing)
    const float mx = wave_max(mine ? ml.x : -__builtin_inff()), w = mine ? __builtin_amdgcn_exp2f(ml.x - mx) : 0.0f;
    const float den = wave_sum(mine && lane < 8 ? w * ml.y : 0.0f), inv = den == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(den);
    f32x4 num = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        if (u > 0 && u * PARTS >= splits) break;
        const int s = p + u * PARTS;
        const float f = __shfl(w, s, WAVE), there = __shfl(mine ? 1.0f : 0.0f, s, WAVE);
        if (there != 0.0f) {
#pragma unroll
            for (int i = 0; i < 4; ++i) num[i] = __builtin_fmaf(f, v[u][i], num[i]);
        }
    }
#pragma unroll
    for (int off = LANES; off < 64; off <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) num[i] += __shfl_xor(num[i], off, WAVE);
    if (p == 0)
        *reinterpret_cast<u32x2*>(out + size_t(row) * D + e) =
            u32x2{f32_to_bf16x2(num[0] * inv, num[1] * inv), f32_to_bf16x2(num[2] * inv, num[3] * inv)};
}

template <int D>
static void launch_join(const TreeArgs& a, hipStream_t st) {
    if (a.splits == 1) return;
    const unsigned rows = unsigned(a.T) * a.hq, fours = (rows + JNT / 64 - 1) / (JNT / 64);
    if (a.splits <= 8)
        attn_tree_join_rows_kernel<D><<<dim3(fours), dim3(JNT), 0, st>>>(a.part, a.out, a.T, a.hq, a.rows, a.splits, a.pos_dev, a.pos0);
    else if (a.splits <= 16)
        attn_tree_join_kernel<D, 16><<<dim3(rows), dim3(JNT), 0, st>>>(a.part, a.out, a.T, a.hq, a.rows, a.splits, a.pos_dev, a.pos0);
    else
        attn_tree_join_kernel<D, 64><<<dim3(rows), dim3(JNT), 0, st>>>(a.part, a.out, a.T, a.hq, a.rows, a.splits, a.pos_dev, a.pos0);
}

}  // namespace scmx
