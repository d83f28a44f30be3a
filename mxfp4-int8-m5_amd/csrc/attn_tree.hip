// Attention of a tree of drafted tokens (1..64 of them) against a KV cache in bf16 or 8 bits (include/scmx_cache.h, scmx_attn_tree).
//
// The tokens' query heads that share a KV head are the rows of one matrix product, so that a cache row is read once for all of
// them: row r is token r / group, head r % group of the group.  A wave owns 16 or 32 rows and walks tiles of 32 keys with a running
// reference (the softmax's maximum), sums in float32 (8 bits: denominators in float64).  Both products are transposed,
//     S^T = K Q^T  (16x16x32 MFMA: rows = keys, columns = queries),   O^T = V^T P^T  (rows = head dimension, columns = queries),
// so that a query is a lane column (lane % 16) in both, its statistics sit in the lanes that need them, and the S^T
// accumulators, converted, are the second product's operand where they are: register 4t + r of lane group g = lane / 16 holds key
// 16t + 4g + r of the tile, and V is read with the same key order.  The contraction over the head dimension may take any order
// too, and takes the one in which a lane's 16-byte load of a K row is its operand.  A lane reads DPL = d / 16 consecutive values of eight V
// rows and turns them in registers (byte permutes); MFMA i then yields head-dimension indexes DPL * row + i.  So nothing
// is staged: no LDS, no barrier in the loop, every wave streams its own keys with the next tile's loads in flight.  Bound by reading
// the cache from some ten thousand rows on (one token, 40000 rows of 8 x 128 in 8 bits: 15.5 us, 5.4 TB/s, and 3.9 the join), by
// latency and two launches below, and with many tokens by a step's chain of products, exponentials and conversions (64 tokens of 32
// heads: a wave's tile takes 1 us).
//
// 8 bits: K codes become bf16 (exact; q stays as it is), the row's scale multiplies the score.  V codes become half precision
// (exact), and the row's scale goes into the weight, w = p * scale, through the exponent: w = exp2(score + log2(scale) - reference).
// Half-precision weights (2^-12) where bf16 ones (2^-9) would double the result's rounding: the denominator is summed from
// p = w / scale, so w's rounding does not cancel.  In bf16 the denominator is summed from the rounded weights (an MFMA with ones),
// and what rounding one dominating weight suffered cancels.
// The reference moves only when a score passes it by some powers of two, so that most tiles need no cross-lane maximum and no rescaling;
// the weights' range (half precision up to 2^15) sets how many.
//
// The keys are cut into ranges, a workgroup of four waves each, whose float32 sums a second kernel joins; a workgroup's waves take its
// tiles in turn and meet in LDS.
#include <math.h>

#include <type_traits>
#include <utility>

#include "../../include/scmx_cache.h"
#include "attn_tree.h"

namespace scmx {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Broadcast of lane N of each row of 16 lanes to the row.
template <int N>
__device__ __forceinline__ float row_lane(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x150 + N, 0xF, 0xF, true));
}
template <typename F, int... E>
__device__ __forceinline__ void for_eight(F&& f, std::integer_sequence<int, E...>) { (f(std::integral_constant<int, E>{}), ...); }

// Byte B of w, a signed number, as the bits of a float.
template <int B>
__device__ __forceinline__ uint32_t byte_f32(uint32_t w) { return __float_as_uint(float(int8_t(w >> (8 * B)))); }

template <int D, int RT, bool EIGHT>
__global__ __launch_bounds__(TNT, D == 256 && !EIGHT ? 1 : 2) void attn_tree_kernel(const TreeArgs a) {
    constexpr int ROWB = EIGHT ? D : 2 * D;   // bytes of a cache row
    constexpr int KL = ROWB / 64;             // 16-byte loads of a lane from a K row
    constexpr int VW = ROWB / 64;             // words of a lane from a V row
    constexpr int DPL = D / 16;               // head-dimension indexes of a lane in V^T, and MFMAs of the second product
    constexpr int ROWS = 16 * RT, SLICES = D / 32, WAVES = TWAVES, NT = TNT;
    constexpr float NEG = -__builtin_inff();
    // how far scores may pass the reference, and where it is put below the largest score (both in powers of two)
    constexpr float PASS = EIGHT ? 6.0f : 8.0f, BELOW = EIGHT ? 8.0f : 0.0f;
    __shared__ float s_o[WAVES][ROWS][D + 4];
    // 8 bits: the denominators are sums of weights over scales, up to 2^14 / 2^-107 each, of any number of rows: tiles' sums in float32,
    // the rest in float64 (30000 rows of 2^-98 overflow float32; the time is the same)
    using Den = std::conditional_t<EIGHT, double, float>;
    __shared__ float s_m[WAVES][ROWS];     // references
    __shared__ Den s_l[WAVES][ROWS];       // denominators

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), ln = lane & 15, g = lane >> 4;
    // blocks of the query rows of one range and KV head run on one XCD, behind one L2
    const int turn = int(blockIdx.x) / (TXCDS * a.blocks), in = int(blockIdx.x) % (TXCDS * a.blocks);
    const int block = in / TXCDS, combo = turn * TXCDS + in % TXCDS;
    if (combo >= a.hk * a.splits) return;
    const int kvh = combo % a.hk, range = combo / a.hk, group = a.hq / a.hk, rows_all = a.T * group;
    const int row0 = block * ROWS;
    const auto token = [&](int r) { return group == 1 ? r : int(__umulhi(uint32_t(r), a.by_group)); };
    const auto out_row = [&](int r) { return size_t(token(r)) * a.hq + size_t(kvh) * group + (r - token(r) * group); };   // of [T, hq]

    const int64_t pos64 = a.pos_dev ? a.pos_dev[0] : a.pos0;
    if (pos64 < 0 || pos64 > int64_t(a.rows) - a.T) {   // (a device-resident position that the host could not see)
        if (range == 0)
            for (int i = tid; i < ROWS * D; i += NT)
                if (row0 + i / D < rows_all) a.out[out_row(row0 + i / D) * D + i % D] = 0;
        return;
    }
    const int pos = int(pos64), n = pos + a.T, tiles = tiles_of(n);
    const int per = range_tiles(n, a.splits);
    const int first = range * per, last = min(tiles, first + per);
    if (first >= last) return;   // an empty range: the join knows
    const bool whole = per >= tiles;

    const uint8_t* kb = a.k + size_t(kvh) * a.rows * ROWB;
    const uint8_t* vb = a.v + size_t(kvh) * a.rows * ROWB;
    u32x4 kr[2][KL];
    uint32_t vr[8][VW];
    float sc = 0.0f;   // 8 bits: lanes 0..7 of a row of 16 hold the K scales of the row's eight keys, 8..15 the V scales
    // (The last row stands in for the ones behind it, which are not read.  A branch that spares full tiles the minima costs the loads'
    // overlap: 40000 rows in one range 237 -> 260 us.)
    const auto load_k = [&](int tile) __attribute__((always_inline)) {
        const int base = tile * TKEYS;
        const auto row = [&](int i) { return min(i, n - 1 - base); };
        const uint8_t* kt = kb + size_t(base) * ROWB;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const unsigned at = unsigned(row(16 * h + ln) * ROWB + 16 * g);
#pragma unroll
            for (int u = 0; u < KL; ++u) kr[h][u] = *reinterpret_cast<const u32x4*>(kt + at + 64 * u);
        }
        if constexpr (EIGHT) {
            const float* from = (ln < 8 ? a.ks : a.vs) + size_t(kvh) * a.rows + base;
            sc = from[row(16 * (ln / 4 % 2) + 4 * g + ln % 4)];
        }
    };
    const auto load_v = [&](int tile) __attribute__((always_inline)) {
        const int base = tile * TKEYS;
        const auto row = [&](int i) { return min(i, n - 1 - base); };
        const uint8_t* vt = vb + size_t(base) * ROWB;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint8_t* p = vt + unsigned(row(16 * (e / 4) + 4 * g + e % 4) * ROWB + ROWB / 16 * ln);
            if constexpr (VW == 1) {
                vr[e][0] = *reinterpret_cast<const uint32_t*>(p);
            } else if constexpr (VW == 2) {
                const u32x2 w = *reinterpret_cast<const u32x2*>(p);
                vr[e][0] = w[0];
                vr[e][1] = w[1];
            } else {
#pragma unroll
                for (int u = 0; u < VW / 4; ++u) {
                    const u32x4 w = *reinterpret_cast<const u32x4*>(p + 16 * u);
#pragma unroll
                    for (int i = 0; i < 4; ++i) vr[e][4 * u + i] = w[i];
                }
            }
        }
    };
    // The queries.  32 rows, or rows of 256, come through LDS: read by every wave for itself, as 64-byte pieces of 16 rows an
    // instruction, they held up the first keys by 1.5 us (16 tokens, 300 rows: 10.9 -> 8.9 us); 16 rows of 128 do not (6.6, direct 6.2).
    constexpr bool QLDS = RT > 1 || D > 128;
    constexpr int QPIECES = ROWS * D / 8, QROW = D + 8;   // 16-byte pieces; LDS row in values
    constexpr int QPER = (QPIECES + NT - 1) / NT;         // a thread (the ones left over bring some again)
    __shared__ __attribute__((aligned(16))) uint16_t s_q[QLDS ? ROWS * QROW : 1];
    // slice s of a lane, in K's order
    const auto q_at = [&](int s) { return EIGHT ? 64 * (s / 2) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g; };
    bf16x8 qf[RT][SLICES];
    u32x4 qraw[QPER];
    if constexpr (QLDS) {
#pragma unroll
        for (int i = 0; i < QPER; ++i) {
            const int c = (tid + NT * i) % QPIECES;
            qraw[i] = *reinterpret_cast<const u32x4*>(a.q + out_row(min(row0 + c / (D / 8), rows_all - 1)) * D + c % (D / 8) * 8);
        }
    }
    uint64_t seen[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int i = token(min(row0 + 16 * rt + ln, rows_all - 1));
        seen[rt] = (a.mask ? uint64_t(a.mask[i]) : ~0ull >> (63 - i)) & ~0ull >> (64 - a.T);
    }
    __builtin_amdgcn_sched_barrier(0);
    const int start = first + wave < last ? first + wave : last - 1;   // (a wave without a tile loads one and uses none)
    load_k(start);
    if constexpr (!QLDS) {
        const uint16_t* qp = a.q + out_row(min(row0 + ln, rows_all - 1)) * D;
#pragma unroll
        for (int s = 0; s < SLICES; ++s) qf[0][s] = *reinterpret_cast<const bf16x8*>(qp + q_at(s));
    }
    load_v(start);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (QLDS) {
#pragma unroll
        for (int i = 0; i < QPER; ++i) {
            const int c = (tid + NT * i) % QPIECES;
            *reinterpret_cast<u32x4*>(s_q + c / (D / 8) * QROW + c % (D / 8) * 8) = qraw[i];
        }
        __syncthreads();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int s = 0; s < SLICES; ++s) qf[rt][s] = *reinterpret_cast<const bf16x8*>(s_q + (16 * rt + ln) * QROW + q_at(s));
    }
    f32x4 o[RT][DPL], ones[RT];   // ones: sums of the rounded weights (bf16)
    float m[RT];
    Den l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int i = 0; i < DPL; ++i) o[rt][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        ones[rt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m[rt] = NEG;
        l[rt] = 0;
    }

    // K of the next tile is requested when this one's scores stand, V when its product does: each has the other half of the
    // step to arrive, and no second set of registers.
    for (int tile = first + wave; tile < last; tile += WAVES) {
        const int base = tile * TKEYS, next = min(tile + WAVES, last - 1);
        const bool tail = base > pos - TKEYS;   // the tile reaches into the tree, or past the last row
        // ---- scores
        f32x4 s[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][0] = s[rt][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int sl = 0; sl < SLICES; ++sl)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                bf16x8 kf;
                if constexpr (EIGHT) {
                    const uint32_t w0 = kr[h][sl / 2][2 * (sl & 1)], w1 = kr[h][sl / 2][2 * (sl & 1) + 1];
                    const u32x4 p = {
                        perm(byte_f32<1>(w0), byte_f32<0>(w0), 0x07060302u), perm(byte_f32<3>(w0), byte_f32<2>(w0), 0x07060302u),
                        perm(byte_f32<1>(w1), byte_f32<0>(w1), 0x07060302u), perm(byte_f32<3>(w1), byte_f32<2>(w1), 0x07060302u)};
                    kf = __builtin_bit_cast(bf16x8, p);
                } else {
                    kf = __builtin_bit_cast(bf16x8, kr[h][sl]);
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) s[rt][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[rt][sl], s[rt][h], 0, 0, 0);
            }
        const float scales = sc;
        __builtin_amdgcn_sched_barrier(0);
        load_k(next);
        __builtin_amdgcn_sched_barrier(0);
        // ---- in powers of two; masked
        float x[RT][8], inverse = 0.0f;
        if constexpr (EIGHT) {
            // A row of zeros (scale 0) counts in the denominator alone: it takes a scale below all that matter beside it, so that its score
            // does not set the reference (as 1 it took the bits of rows of 1e-6), and no smaller, so that its weight is not below
            // float32 beside large values.
            const float vscale = scales == 0.0f && ln >= 8 ? 0x1p-80f : scales;
            const float both = ln < 8 ? scales * a.scale : __builtin_amdgcn_logf(vscale);
            inverse = __builtin_amdgcn_rcpf(vscale);
            inverse = inverse == inverse ? inverse : 1.0f;   // (0 times NaN: the nodes that do not see the row)
            for_eight([&](auto e) __attribute__((always_inline)) {
                constexpr int E = decltype(e)::value;
                const float k = row_lane<E>(both), lv = row_lane<8 + E>(both);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) x[rt][E] = __builtin_fmaf(s[rt][E / 4][E % 4], k, lv);
            }, std::make_integer_sequence<int, 8>{});
        } else {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[rt][e] = s[rt][e / 4][e % 4] * a.scale;
        }
        if (tail) {
            const int below = pos - base;   // rows of the tile before the tree (negative: rows of the tree before the tile, up to 63)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {   // bit k: key k of the tile is seen; shifted to the lane's first key
                const uint32_t window = uint32_t(below > 0 ? seen[rt] << below | ((1ull << below) - 1) : seen[rt] >> -below) >> (4 * g);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[rt][e] = window & (1u << (16 * (e / 4) + e % 4)) ? x[rt][e] : NEG;
            }
        }
        // ---- the reference moves where a score passes it
        bool any = false;
        float top[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            top[rt] = x[rt][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) top[rt] = fmaxf(top[rt], x[rt][e]);
            any |= top[rt] > m[rt] + (BELOW + PASS);
        }
        if (__builtin_amdgcn_ballot_w64(any)) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float t0 = fmaxf(top[rt], __shfl_xor(top[rt], 16, WAVE));
                t0 = fmaxf(t0, __shfl_xor(t0, 32, WAVE));
                // (each query by its own scores alone: no other query's change what it gets)
                const float mn = t0 > m[rt] + (BELOW + PASS) ? t0 - BELOW : m[rt];
                const float alpha = mn == NEG ? 1.0f : __builtin_amdgcn_exp2f(m[rt] - mn);
                m[rt] = mn;
                l[rt] *= alpha;
#pragma unroll
                for (int r = 0; r < 4; ++r) ones[rt][r] *= alpha;
#pragma unroll
                for (int i = 0; i < DPL; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[rt][i][r] *= alpha;
            }
        }
        // ---- weights
        u32x4 pf[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float shift = m[rt] == NEG ? 0.0f : m[rt];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[rt][e] = __builtin_amdgcn_exp2f(x[rt][e] - shift);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (EIGHT) {
                    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
                    pf[rt][e] = __builtin_bit_cast(uint32_t, f16x2{_Float16(x[rt][2 * e]), _Float16(x[rt][2 * e + 1])});
                } else {
                    pf[rt][e] = f32_to_bf16x2(x[rt][2 * e], x[rt][2 * e + 1]);
                }
            }
        }
        if constexpr (EIGHT) {
            float eight[RT] = {};   // (below 2^124)
            for_eight([&](auto e) __attribute__((always_inline)) {
                constexpr int E = decltype(e)::value;
                const float iv = row_lane<8 + E>(inverse);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) eight[rt] = __builtin_fmaf(x[rt][E], iv, eight[rt]);
            }, std::make_integer_sequence<int, 8>{});
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) l[rt] += double(eight[rt]);
        }
        // ---- the tree's rows in bf16: a row that is not finite must not reach (0 times infinity) the queries that do not see it
        if (!EIGHT && tail) {
            uint32_t odd[8], any_odd = 0;   // not zero: some value of the row is an infinity or NaN (the exponent's carry)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int j = base + 16 * (e / 4) + 4 * g + e % 4 - pos;
                odd[e] = 0;
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    odd[e] |= (vr[e][w] & 0x7F807F80u) + 0x00800080u;
                    vr[e][w] = j < a.T ? vr[e][w] : 0;   // behind the last row: a copy of that
                }
                odd[e] = j >= 0 && j < a.T ? odd[e] & 0x80008000u : 0;
                any_odd |= odd[e];
            }
            uint32_t bad = 0;
            if (__builtin_amdgcn_ballot_w64(any_odd != 0)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint64_t b = __builtin_amdgcn_ballot_w64(odd[e] != 0);
                    const uint32_t of = uint32_t((b & 0xFFFFu) != 0) | uint32_t((b >> 16 & 0xFFFFu) != 0) << 1 |
                                        uint32_t((b >> 32 & 0xFFFFu) != 0) << 2 | uint32_t((b >> 48) != 0) << 3;
                    bad |= of << (4 * e);
#pragma unroll
                    for (int w = 0; w < VW; ++w) vr[e][w] = of >> g & 1 ? 0 : vr[e][w];
                }
            }
            if (bad) {   // rare: those rows by hand, for the queries that see them; their weights through LDS, which is free here
                float* const w = &s_o[wave][0][0];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[(rt * 32 + 4 * e + g) * 16 + ln] = x[rt][e];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                for (; bad; bad &= bad - 1) {
                    const int at = __builtin_ctz(bad), key = base + 16 * (at / 16) + 4 * (at % 4) + at / 4 % 4;
                    const uint16_t* row = reinterpret_cast<const uint16_t*>(vb + size_t(key) * ROWB) + DPL * 4 * g;
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        const float p = w[(rt * 32 + at) * 16 + ln];
                        if (seen[rt] >> (key - pos) & 1) {
#pragma unroll
                            for (int r = 0; r < 4; ++r)
#pragma unroll
                                for (int i = 0; i < DPL; ++i) o[rt][i][r] = __builtin_fmaf(p, bf16_to_f32(row[DPL * r + i]), o[rt][i][r]);
                        }
                    }
                }
            }
        }
        // ---- O^T += V^T P^T
        if constexpr (!EIGHT) {
            const u32x4 one = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
                ones[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, one), __builtin_bit_cast(bf16x8, pf[rt]),
                                                                   ones[rt], 0, 0, 0);
        }
        uint32_t pairs[2][4];   // 8 bits: bytes 0, 1 and 2, 3 of a word of two rows, side by side
#pragma unroll
        for (int i = 0; i < DPL; ++i) {
            u32x4 w;
            if constexpr (EIGHT) {
                // half precision 1024 + 128 + code: the code biased by 128 beside the byte 0x64
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (i % 4 == 0) {
                        const uint32_t lo = vr[2 * e][i / 4] ^ 0x80808080u, hi = vr[2 * e + 1][i / 4] ^ 0x80808080u;
                        pairs[0][e] = perm(hi, lo, 0x05010400u);
                        pairs[1][e] = perm(hi, lo, 0x07030602u);
                    }
                    const uint32_t two = perm(0x64646464u, pairs[i % 4 / 2][e], i % 2 ? 0x04030402u : 0x04010400u);
                    const half2_t biased = __builtin_bit_cast(half2_t, two);
                    w[e] = __builtin_bit_cast(uint32_t, half2_t(biased - half2_t{_Float16(1152.0f), _Float16(1152.0f)}));
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    o[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w), __builtin_bit_cast(f16x8, pf[rt]),
                                                                      o[rt][i], 0, 0, 0);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = perm(vr[2 * e + 1][i / 2], vr[2 * e][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    o[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, pf[rt]),
                                                                       o[rt][i], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_v(next);
        __builtin_amdgcn_sched_barrier(0);
    }

    // ---- the waves meet: their references first, so that what they leave in LDS only has to be added
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if constexpr (EIGHT) {
            l[rt] += __shfl_xor(l[rt], 16, WAVE);
            l[rt] += __shfl_xor(l[rt], 32, WAVE);
        } else {
            l[rt] = ones[rt][0];
        }
        if (g == 0) {
            s_m[wave][16 * rt + ln] = m[rt];
            s_l[wave][16 * rt + ln] = l[rt];
        }
    }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = 16 * rt + ln;
        float mw[WAVES], mx = NEG;
        Den lw[WAVES], sum = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            mw[w] = s_m[w][r];
            lw[w] = s_l[w][r];
            mx = fmaxf(mx, mw[w]);
        }
#pragma unroll
        for (int w = 0; w < WAVES; ++w)   // (l is 0 of a wave whose keys the query does not see)
            if (lw[w] != 0) {
                if constexpr (EIGHT) sum = __builtin_fma(double(__builtin_amdgcn_exp2f(mw[w] - mx)), lw[w], sum);
                else sum = __builtin_fmaf(__builtin_amdgcn_exp2f(mw[w] - mx), lw[w], sum);
            }
        float f = l[rt] == 0 ? 0.0f : __builtin_amdgcn_exp2f(m[rt] - mx);
        if (EIGHT && sum > 0x1p100) {   // rows of very small values: the sums in other units
            sum *= 0x1p-64;
            mx += 64.0f;
#pragma unroll
            for (int i = 0; i < DPL; ++i)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) o[rt][i][r4] *= 0x1p-64f;
        }
        const float den = float(sum);
        if (whole) f *= den == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(den);   // (0: nothing was seen)
        else if (wave == 0 && g == 0 && row0 + r < rows_all)
            *reinterpret_cast<float2*>(a.part + size_t(a.T) * a.hq * a.splits * D +
                                       2 * (out_row(row0 + r) * a.splits + range)) = float2{mx, den};
        if (row0 + r < rows_all) {
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
#pragma unroll
                for (int i = 0; i < DPL; i += 4)
                    *reinterpret_cast<f32x4*>(&s_o[wave][r][DPL * (4 * g + q4) + i]) =
                        f32x4{o[rt][i][q4] * f, o[rt][i + 1][q4] * f, o[rt][i + 2][q4] * f, o[rt][i + 3][q4] * f};
        }
    }
    __syncthreads();
    for (int c = tid; c < ROWS * (D / 4); c += NT) {
        const int r = c / (D / 4), e = c % (D / 4) * 4;
        if (row0 + r >= rows_all) break;
        f32x4 v[WAVES];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v[w] = *reinterpret_cast<const f32x4*>(&s_o[w][r][e]);
#pragma unroll
        for (int w = 1; w < WAVES; ++w)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[0][i] += v[w][i];
        const size_t at = out_row(row0 + r);
        if (whole) *reinterpret_cast<u32x2*>(a.out + at * D + e) = u32x2{f32_to_bf16x2(v[0][0], v[0][1]), f32_to_bf16x2(v[0][2], v[0][3])};
        else *reinterpret_cast<f32x4*>(a.part + (at * a.splits + range) * D + e) = v[0];
    }
}

template <int D, int RT>
static void launch_tree(const TreeArgs& a, hipStream_t st) {
    const unsigned combos = unsigned(a.hk) * a.splits, grid = (combos + TXCDS - 1) / TXCDS * TXCDS * a.blocks;
    if (a.ks) attn_tree_kernel<D, RT, true><<<dim3(grid), dim3(TNT), 0, st>>>(a);
    else attn_tree_kernel<D, RT, false><<<dim3(grid), dim3(TNT), 0, st>>>(a);
    launch_join<D>(a, st);
}

}  // namespace scmx

using namespace scmx;

// 16-row blocks of queries a wave: two where there are that many rows and its registers hold them.
static int tree_blocks(int qrows, int d) { return qrows <= 16 || d == 256 ? 1 : 2; }

extern "C" int scmx_attn_tree_splits(int T, int n, int hq, int hk, int d) {
    if (T < 1 || T > 64 || n < 1 || hq < 1 || hk < 1 || hq > 65535 || hq % hk || (d != 64 && d != 128 && d != 256)) return 1;
    const int qrows = T * (hq / hk), rt = tree_blocks(qrows, d), tiles = tiles_of(n);
    if (tiles <= TONE) return 1;
    // A workgroup a CU, a tile a wave; up to 32 ranges of one tile a wave are 16 of two instead, whose join reads half as much.  That pays
    // for 32 query rows of 128 (16 tokens of 16:8 x 128, 16 ranges / a tile a wave: 94 tiles 10.9 / 11.2 us, 128 tiles bf16 12.4 / 13.0,
    // 65 tiles 10.7 / 10.5), and costs fewer or narrower rows 0.1 to 0.4 us (94 tiles, one token of 16:8 x 128 8.5 / 8.4, of 14:2 x 64
    // 7.1 / 6.8), one token over bf16 rows of 256 up to 1.6 (128 tiles 15.2 / 13.6).
    const int64_t most = 256 / (int64_t(hk) * ((qrows + 16 * rt - 1) / (16 * rt)));
    const int even = (tiles + TWAVES - 1) / TWAVES, ranges = even > 16 && even <= 32 ? 16 : even < 64 ? even : 64;
    return most < 1 ? 1 : ranges < most ? ranges : int(most);
}

extern "C" int scmx_attn_tree(const uint16_t* q, const void* kcache, const void* vcache, const float* kscale, const float* vscale,
                              const int64_t* mask, const int64_t* pos_dev, int64_t pos0, uint16_t* out, int T, int hq, int hk, int d,
                              int cache_rows, float scale, float* workspace, int splits, void* stream) {
    if (!q || !kcache || !vcache || !out || !kscale != !vscale) {
        set_error("attn_tree: null pointer argument (an 8-bit cache has both scales, a bf16 one none)");
        return SCMX_ERR_ARG;
    }
    if (T < 1 || T > 64 || hq < 1 || hk < 1 || hq > 65535 || hq % hk || hq / hk > 4096 || cache_rows < T) {
        set_error("attn_tree: need 1..64 nodes, hq %% hk == 0, up to 4096 query heads a KV head and a cache that holds the tree "
                  "(T=%d hq=%d hk=%d rows=%d)", T, hq, hk, cache_rows);
        return SCMX_ERR_ARG;
    }
    if (d != 64 && d != 128 && d != 256) {
        set_error("attn_tree: head dim must be 64, 128 or 256 (d=%d)", d);
        return SCMX_ERR_ARG;
    }
    if (!pos_dev && (pos0 < 0 || pos0 > int64_t(cache_rows) - T)) {
        set_error("attn_tree: %d rows from %lld on do not fit a cache of %d rows", T, (long long)pos0, cache_rows);
        return SCMX_ERR_ARG;
    }
    if (!(fabsf(scale * 1.4426950408889634f) <= 3.4028234e38f)) {   // (the kernel works in powers of two)
        set_error("attn_tree: scale must be finite, times log2 e too");
        return SCMX_ERR_ARG;
    }
    if ((uintptr_t(q) | uintptr_t(kcache) | uintptr_t(vcache) | uintptr_t(out)) % 16) {
        set_error("attn_tree: q, out and the caches must be 16-byte aligned");
        return SCMX_ERR_ARG;
    }
    if (splits < 1 || splits > 64 || (splits > 1 && (!workspace || uintptr_t(workspace) % 16))) {
        set_error("attn_tree: splits must be 1..64 and need a 16-byte aligned workspace of splits * T * hq * (d + 2) floats");
        return SCMX_ERR_ARG;
    }
    const int qrows = T * (hq / hk);
    const uint32_t by_group = uint32_t(((uint64_t(1) << 32) + hq / hk - 1) / uint64_t(hq / hk));
    TreeArgs a{q, static_cast<const uint8_t*>(kcache), static_cast<const uint8_t*>(vcache), kscale, vscale, mask, pos_dev, pos0, out,
               workspace, T, hq, hk, cache_rows, splits, 0, by_group, scale * 1.4426950408889634f};
    const int rt = tree_blocks(qrows, d);
    a.blocks = (qrows + 16 * rt - 1) / (16 * rt);
    const hipStream_t st = (hipStream_t)stream;
    const auto go = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        if (rt == 1) launch_tree<D, 1>(a, st);
        else if constexpr (D < 256) launch_tree<D, 2>(a, st);
    };
    if (d == 64) go(std::integral_constant<int, 64>{});
    else if (d == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
    return check_launch("attn_tree");
}
