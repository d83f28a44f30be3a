// Attention of a tree of drafted tokens (1..64 of them) against a KV cache in bf16 or 8 bits (include/scmx_cache.h, scmx_attn_tree).
//
// The tokens' query heads that share a KV head are the rows of one matrix product, so that a cache row is read once for all of
// them: row r is token r / group, head r % group of the group.  A wave owns 16, 32 or 64 rows and walks tiles of 32 keys with a running
// reference (the softmax's maximum), sums in float32.  Both products are transposed,
//     S^T = K Q^T  (16x16x32 MFMA: rows = keys, columns = queries),   O^T = V^T P^T  (rows = head dimension, columns = queries),
// so that a query is a lane column (lane % 16) in both, its statistics sit in the lanes that need them, and the S^T
// accumulators, converted, are the second product's operand where they are: register 4t + r of lane group g = lane / 16 holds key
// 16t + 4g + r of the tile, and V is read with the same key order.  The contraction over the head dimension may take any order
// too, and takes the one in which a lane's 16-byte load of a K row is its operand.  A lane reads DPL = d / 16 consecutive values of eight V
// rows and turns them in registers (byte permutes); MFMA i then yields head-dimension indexes DPL * row + i.  So nothing
// is staged: no LDS, no barrier in the loop, every wave streams its own keys with the next tile's loads in flight.
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

#include "../../include/scmx_cache.h"
#include "scmx_common.h"

namespace scmx {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));   // scales: aligned as floats

constexpr int TNT = 256, TWAVES = TNT / 64, TKEYS = 32, TXCDS = 8;
constexpr int TTILES_MIN = 8;   // tiles a range has at least (two a wave), where there are that many

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
    float* part;      // [splits][T hq][d] sums, then [splits][T hq][2]: reference, denominator
    int T, hq, hk, rows, splits, blocks;   // blocks: of query rows
    float scale;      // times log2 e
};

// The ranges of a context of n keys in all: tiles each, and how many of them have any.
static __device__ __host__ inline int range_tiles(int n, int splits) {
    const int tiles = (n + TKEYS - 1) / TKEYS, even = (tiles + splits - 1) / splits;
    return even > TTILES_MIN ? even : TTILES_MIN;
}

template <int D, int RT, bool EIGHT>
struct Tree {
    static constexpr int ROWB = EIGHT ? D : 2 * D;   // bytes of a cache row
    static constexpr int KL = ROWB / 64;             // 16-byte loads of a lane from a K row
    static constexpr int VW = ROWB / 64;             // words of a lane from a V row
    static constexpr int DPL = D / 16;               // head-dimension indexes of a lane in V^T, and MFMAs of the second product
    static constexpr int ROWS = 16 * RT;
    // What one tile of keys is loaded into.
    struct Raw {
        u32x4 k[2][KL];
        uint32_t v[8][VW];
        float ks[8], vs[8];
    };
};

// v_cvt_f32 of byte B of w as a signed number, as the bits of a float.
template <int B>
__device__ __forceinline__ uint32_t byte_f32(uint32_t w) { return __float_as_uint(float(int8_t(w >> (8 * B)))); }

template <int D, int RT, bool EIGHT>
__global__ __launch_bounds__(TNT, 1) void attn_tree_kernel(const TreeArgs a) {
    using W = Tree<D, RT, EIGHT>;
    constexpr int ROWB = W::ROWB, KL = W::KL, VW = W::VW, DPL = W::DPL, SLICES = D / 32;
    constexpr float NEG = -__builtin_inff();
    // how far scores may pass the reference, and where it is put below the largest score (both in powers of two)
    constexpr float PASS = EIGHT ? 6.0f : 8.0f, BELOW = EIGHT ? 8.0f : 0.0f;
    __shared__ float s_o[TWAVES][W::ROWS][D + 4];
    __shared__ float s_m[TWAVES][W::ROWS], s_l[TWAVES][W::ROWS];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), ln = lane & 15, g = lane >> 4;
    // blocks of the query rows of one range and KV head run on one XCD, behind one L2
    const int turn = int(blockIdx.x) / (TXCDS * a.blocks), in = int(blockIdx.x) % (TXCDS * a.blocks);
    const int block = in / TXCDS, combo = turn * TXCDS + in % TXCDS;
    if (combo >= a.hk * a.splits) return;
    const int kvh = combo % a.hk, range = combo / a.hk, group = a.hq / a.hk, rows_all = a.T * group;
    const int row0 = block * W::ROWS;
    const auto out_row = [&](int r) { return size_t(r / group) * a.hq + size_t(kvh) * group + r % group; };   // of [T, hq]

    const int64_t pos64 = a.pos_dev ? a.pos_dev[0] : a.pos0;
    if (pos64 < 0 || pos64 > int64_t(a.rows) - a.T) {   // (a device-resident position that the host could not see)
        if (range == 0)
            for (int i = tid; i < W::ROWS * D; i += TNT)
                if (row0 + i / D < rows_all) a.out[out_row(row0 + i / D) * D + i % D] = 0;
        return;
    }
    const int pos = int(pos64), n = pos + a.T, tiles = (n + TKEYS - 1) / TKEYS;
    const int per = range_tiles(n, a.splits);
    const int first = range * per, last = min(tiles, first + per);
    if (first >= last) return;   // an empty range: the join knows
    const bool whole = per >= tiles;

    bf16x8 qf[RT][SLICES];
    uint64_t seen[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = min(row0 + 16 * rt + ln, rows_all - 1);
        const uint16_t* qp = a.q + out_row(r) * D;
#pragma unroll
        for (int s = 0; s < SLICES; ++s)
            qf[rt][s] = *reinterpret_cast<const bf16x8*>(qp + (EIGHT ? 64 * (s / 2) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g));
        const int i = r / group;
        seen[rt] = a.mask ? uint64_t(a.mask[i]) : ~0ull >> (63 - i);
    }
    f32x4 o[RT][DPL], ones[RT];   // ones: sums of the rounded weights (bf16)
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int i = 0; i < DPL; ++i) o[rt][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        ones[rt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m[rt] = NEG;
        l[rt] = 0.0f;
    }

    const uint8_t* kb = a.k + size_t(kvh) * a.rows * ROWB;
    const uint8_t* vb = a.v + size_t(kvh) * a.rows * ROWB;
    const float* ksb = EIGHT ? a.ks + size_t(kvh) * a.rows : nullptr;
    const float* vsb = EIGHT ? a.vs + size_t(kvh) * a.rows : nullptr;

    auto load_at = [&](typename W::Raw& t, int base, auto row) __attribute__((always_inline)) {   // row(i): row i of the tile, as one that is there
        const uint8_t* kt = kb + size_t(base) * ROWB;
        const uint8_t* vt = vb + size_t(base) * ROWB;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int u = 0; u < KL; ++u) t.k[h][u] = *reinterpret_cast<const u32x4*>(kt + unsigned(row(16 * h + ln) * ROWB + 64 * u + 16 * g));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint8_t* p = vt + unsigned(row(16 * (e / 4) + 4 * g + e % 4) * ROWB + ROWB / 16 * ln);
            if constexpr (VW == 1) {
                t.v[e][0] = *reinterpret_cast<const uint32_t*>(p);
            } else if constexpr (VW == 2) {
                const u32x2 w = *reinterpret_cast<const u32x2*>(p);
                t.v[e][0] = w[0];
                t.v[e][1] = w[1];
            } else {
#pragma unroll
                for (int u = 0; u < VW / 4; ++u) {
                    const u32x4 w = *reinterpret_cast<const u32x4*>(p + 16 * u);
#pragma unroll
                    for (int i = 0; i < 4; ++i) t.v[e][4 * u + i] = w[i];
                }
            }
        }
    };
    auto load = [&](typename W::Raw& t, int tile) __attribute__((always_inline)) {
        const int base = tile * TKEYS;
        if (base + TKEYS <= n) {
            load_at(t, base, [](int i) { return i; });
            if constexpr (EIGHT) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f32x4u a4 = *reinterpret_cast<const f32x4u*>(ksb + base + 16 * h + 4 * g), b4 = *reinterpret_cast<const f32x4u*>(vsb + base + 16 * h + 4 * g);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        t.ks[4 * h + r] = a4[r];
                        t.vs[4 * h + r] = b4[r];
                    }
                }
            }
        } else {   // the last tile: rows behind the last one are not read
            const auto there = [&](int i) { return min(i, n - 1 - base); };
            load_at(t, base, there);
            if constexpr (EIGHT) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int at = base + there(16 * (e / 4) + 4 * g + e % 4);
                    t.ks[e] = ksb[at];
                    t.vs[e] = vsb[at];
                }
            }
        }
    };

    auto work = [&](typename W::Raw& t, int tile, auto tail) __attribute__((always_inline)) {
        constexpr bool TAIL = decltype(tail)::value;   // the tile reaches into the tree, or past the last row
        const int base = tile * TKEYS;
        // ---- scores, in powers of two
        float x[RT][8], iv[8];
        {
            f32x4 s[RT][2];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) s[rt][0] = s[rt][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int sl = 0; sl < SLICES; ++sl)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    bf16x8 kf;
                    if constexpr (EIGHT) {
                        const uint32_t w0 = t.k[h][sl / 2][2 * (sl & 1)], w1 = t.k[h][sl / 2][2 * (sl & 1) + 1];
                        const u32x4 p = {perm(byte_f32<1>(w0), byte_f32<0>(w0), 0x07060302u), perm(byte_f32<3>(w0), byte_f32<2>(w0), 0x07060302u),
                                         perm(byte_f32<1>(w1), byte_f32<0>(w1), 0x07060302u), perm(byte_f32<3>(w1), byte_f32<2>(w1), 0x07060302u)};
                        kf = __builtin_bit_cast(bf16x8, p);
                    } else {
                        kf = __builtin_bit_cast(bf16x8, t.k[h][sl]);
                    }
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) s[rt][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[rt][sl], s[rt][h], 0, 0, 0);
                }
            float kscale[8], lv[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                kscale[e] = EIGHT ? t.ks[e] * a.scale : a.scale;
                if constexpr (EIGHT) {
                    // a row of zeros (scale 0) counts in the denominator alone
                    t.vs[e] = t.vs[e] == 0.0f ? 1.0f : t.vs[e];
                    lv[e] = __builtin_amdgcn_logf(t.vs[e]);
                    iv[e] = __builtin_amdgcn_rcpf(t.vs[e]);
                    if constexpr (TAIL) iv[e] = iv[e] == iv[e] ? iv[e] : 1.0f;   // (0 times NaN: the nodes that do not see the row)
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[rt][e] = EIGHT ? __builtin_fmaf(s[rt][e / 4][e % 4], kscale[e], lv[e]) : s[rt][e / 4][e % 4] * kscale[e];
                    if constexpr (TAIL) {
                        const int key = base + 16 * (e / 4) + 4 * g + e % 4, j = key - pos;
                        const bool vis = j < 0 || (j < a.T && (seen[rt] >> (j & 63) & 1));
                        x[rt][e] = vis ? x[rt][e] : NEG;
                    }
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
            for (int e = 0; e < 8; ++e) {
                x[rt][e] = __builtin_amdgcn_exp2f(x[rt][e] - shift);
                if constexpr (EIGHT) l[rt] = __builtin_fmaf(x[rt][e], iv[e], l[rt]);
            }
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
        // ---- the tree's rows in bf16: a row that is not finite must not reach (0 times infinity) the queries that do not see it
        if constexpr (TAIL && !EIGHT) {
            uint32_t bad = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int j = base + 16 * (e / 4) + 4 * g + e % 4 - pos;
                bool odd = false;
#pragma unroll
                for (int w = 0; w < VW; ++w) odd |= (t.v[e][w] & 0x7F80u) == 0x7F80u || (t.v[e][w] & 0x7F800000u) == 0x7F800000u;
                const bool gone = j >= a.T;   // behind the last row: a copy of that
                const uint64_t b = __builtin_amdgcn_ballot_w64(odd && j >= 0 && !gone);
                const uint32_t of = uint32_t((b & 0xFFFFu) != 0) | uint32_t((b >> 16 & 0xFFFFu) != 0) << 1 | uint32_t((b >> 32 & 0xFFFFu) != 0) << 2 |
                                    uint32_t((b >> 48) != 0) << 3;
                bad |= of << (4 * e);
                if (gone || (of >> g & 1)) {
#pragma unroll
                    for (int w = 0; w < VW; ++w) t.v[e][w] = 0;
                }
            }
            if (bad) {   // rare: those rows by hand, for the queries that see them; their weights through LDS, which is free here
                float* const w = &s_o[wave][0][0];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[(rt * 32 + 4 * e + g) * 16 + ln] = x[rt][e];
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
                ones[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, one), __builtin_bit_cast(bf16x8, pf[rt]), ones[rt], 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < DPL; ++i) {
            u32x4 w;
            if constexpr (EIGHT) {
                // bytes i of two rows, biased by 128, beside 0x64: half precision 1024 + 128 + code
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t lo = t.v[2 * e][i / 4] ^ 0x80808080u, hi = t.v[2 * e + 1][i / 4] ^ 0x80808080u;
                    const uint32_t two = perm(hi, lo, 0x0C000C00u | uint32_t(i % 4) | uint32_t(4 + i % 4) << 16) | 0x64006400u;
                    w[e] = __builtin_bit_cast(uint32_t, half2_t(__builtin_bit_cast(half2_t, two) - half2_t{_Float16(1152.0f), _Float16(1152.0f)}));
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    o[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w), __builtin_bit_cast(f16x8, pf[rt]), o[rt][i], 0, 0, 0);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = perm(t.v[2 * e + 1][i / 2], t.v[2 * e][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    o[rt][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, pf[rt]), o[rt][i], 0, 0, 0);
            }
        }
    };
    typename W::Raw even, odd;
    int tile = first + wave;
    if (tile < last) load(even, tile);
    const int full = min(last, pos / TKEYS);   // tiles below this one are rows that every node sees
    while (tile + TWAVES < full) {
        load(odd, tile + TWAVES);
        work(even, tile, std::false_type{});
        tile += 2 * TWAVES;
        if (tile < last) load(even, tile);
        work(odd, tile - TWAVES, std::false_type{});
    }
    for (; tile < last; tile += TWAVES) {   // up to one more of those, and the ones that reach into the tree
        if (tile + TWAVES < last) load(odd, tile + TWAVES);
        work(even, tile, std::true_type{});
        even = odd;
    }

    // ---- the waves meet
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if constexpr (EIGHT) {
            l[rt] += __shfl_xor(l[rt], 16, WAVE);
            l[rt] += __shfl_xor(l[rt], 32, WAVE);
        } else {
            l[rt] = ones[rt][0];
        }
        const int r = 16 * rt + ln;
        if (g == 0) {
            s_m[wave][r] = m[rt];
            s_l[wave][r] = l[rt];
        }
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
#pragma unroll
            for (int i = 0; i < DPL; i += 4)
                *reinterpret_cast<f32x4*>(&s_o[wave][r][DPL * (4 * g + q4) + i]) = f32x4{o[rt][i][q4], o[rt][i + 1][q4], o[rt][i + 2][q4], o[rt][i + 3][q4]};
    }
    __syncthreads();
    for (int c = tid; c < W::ROWS * (D / 4); c += TNT) {
        const int r = c / (D / 4), e = c % (D / 4) * 4;
        if (row0 + r >= rows_all) break;
        float mx = s_m[0][r];
#pragma unroll
        for (int w = 1; w < TWAVES; ++w) mx = fmaxf(mx, s_m[w][r]);
        f32x4 num = {0.0f, 0.0f, 0.0f, 0.0f};
        float den = 0.0f;
#pragma unroll
        for (int w = 0; w < TWAVES; ++w) {
            if (s_l[w][r] == 0.0f) continue;   // a wave whose keys the query does not see
            const float f = __builtin_amdgcn_exp2f(s_m[w][r] - mx);
            const f32x4 v = *reinterpret_cast<const f32x4*>(&s_o[w][r][e]);
#pragma unroll
            for (int i = 0; i < 4; ++i) num[i] = __builtin_fmaf(f, v[i], num[i]);
            den = __builtin_fmaf(f, s_l[w][r], den);
        }
        const size_t at = out_row(row0 + r);
        if (whole) {
            const float inv = den == 0.0f ? 0.0f : 1.0f / den;   // (0: nothing was seen)
            const u32x2 w = {f32_to_bf16x2(num[0] * inv, num[1] * inv), f32_to_bf16x2(num[2] * inv, num[3] * inv)};
            *reinterpret_cast<u32x2*>(a.out + at * D + e) = w;
        } else {
            const size_t all = size_t(a.T) * a.hq, slot = size_t(range) * all + at;
            *reinterpret_cast<f32x4*>(a.part + slot * D + e) = num;
            if (e == 0) {
                float* ml = a.part + size_t(a.splits) * all * D + 2 * slot;
                ml[0] = mx;
                ml[1] = den;
            }
        }
    }
}

// Joins the ranges of each row of [T, hq]: D / 4 lanes a row.
template <int D>
__global__ __launch_bounds__(TNT) void attn_tree_join_kernel(const float* __restrict__ part, uint16_t* __restrict__ out, int T, int hq, int rows,
                                                             int splits, const int64_t* pos_dev, int64_t pos0) {
    const int64_t pos = pos_dev ? pos_dev[0] : pos0;
    if (pos < 0 || pos > int64_t(rows) - T) return;   // zeros, written
    const int n = int(pos) + T, per = range_tiles(n, splits), tiles = (n + TKEYS - 1) / TKEYS, ranges = (tiles + per - 1) / per;
    const size_t all = size_t(T) * hq, row = size_t(blockIdx.x) * (TNT / (D / 4)) + threadIdx.x / (D / 4);
    if (ranges == 1 || row >= all) return;
    const int e = threadIdx.x % (D / 4) * 4;
    const float* ml = part + size_t(splits) * all * D + 2 * row;
    constexpr float NEG = -__builtin_inff();
    float mx = NEG;
    for (int s = 0; s < ranges; ++s) mx = fmaxf(mx, ml[2 * s * all]);
    f32x4 num = {0.0f, 0.0f, 0.0f, 0.0f};
    float den = 0.0f;
    for (int s = 0; s < ranges; ++s) {
        const float l = ml[2 * s * all + 1], w = __builtin_amdgcn_exp2f(ml[2 * s * all] - mx);
        const f32x4 v = *reinterpret_cast<const f32x4*>(part + (s * all + row) * D + e);
        if (l == 0.0f) continue;   // a range of which the query sees nothing
#pragma unroll
        for (int i = 0; i < 4; ++i) num[i] = __builtin_fmaf(w, v[i], num[i]);
        den = __builtin_fmaf(w, l, den);
    }
    const float inv = den == 0.0f ? 0.0f : 1.0f / den;
    const u32x2 w = {f32_to_bf16x2(num[0] * inv, num[1] * inv), f32_to_bf16x2(num[2] * inv, num[3] * inv)};
    *reinterpret_cast<u32x2*>(out + row * D + e) = w;
}

template <int D, int RT>
static void launch_tree(const TreeArgs& a, hipStream_t st) {
    const unsigned combos = unsigned(a.hk) * a.splits, grid = (combos + TXCDS - 1) / TXCDS * TXCDS * a.blocks;
    if (a.ks) attn_tree_kernel<D, RT, true><<<dim3(grid), dim3(TNT), 0, st>>>(a);
    else attn_tree_kernel<D, RT, false><<<dim3(grid), dim3(TNT), 0, st>>>(a);
    if (a.splits > 1) {
        constexpr int PER = TNT / (D / 4);
        attn_tree_join_kernel<D><<<dim3((unsigned(a.T) * a.hq + PER - 1) / PER), dim3(TNT), 0, st>>>(a.part, a.out, a.T, a.hq, a.rows, a.splits, a.pos_dev,
                                                                                                  a.pos0);
    }
}

}  // namespace scmx

using namespace scmx;

extern "C" int scmx_attn_tree(const uint16_t* q, const void* kcache, const void* vcache, const float* kscale, const float* vscale,
                              const int64_t* mask, const int64_t* pos_dev, int64_t pos0, uint16_t* out, int T, int hq, int hk, int d,
                              int cache_rows, float scale, float* workspace, int splits, void* stream) {
    if (!q || !kcache || !vcache || !out || !kscale != !vscale) {
        set_error("attn_tree: null pointer argument (an 8-bit cache has both scales, a bf16 one none)");
        return SCMX_ERR_ARG;
    }
    if (T < 1 || T > 64 || hq < 1 || hk < 1 || hq > 65535 || hq % hk || cache_rows < T) {
        set_error("attn_tree: need 1..64 nodes, hq %% hk == 0 and a cache that holds the tree (T=%d hq=%d hk=%d rows=%d)", T, hq, hk, cache_rows);
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
    if (!(scale >= -3.0e38f && scale <= 3.0e38f)) {
        set_error("attn_tree: scale must be finite");
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
    TreeArgs a{q, static_cast<const uint8_t*>(kcache), static_cast<const uint8_t*>(vcache), kscale, vscale, mask, pos_dev, pos0, out, workspace,
               T, hq, hk, cache_rows, splits, 0, scale * 1.4426950408889634f};
    // query rows a wave: as many as there are, up to what its registers hold (64 rows of 128, 32 of 256)
    const int rt = qrows <= 16 ? 1 : qrows <= 32 || d == 256 ? 2 : 4;
    a.blocks = (qrows + 16 * rt - 1) / (16 * rt);
    const hipStream_t st = (hipStream_t)stream;
    const auto go = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        if (rt == 1) launch_tree<D, 1>(a, st);
        else if (rt == 2) launch_tree<D, 2>(a, st);
        else if constexpr (D < 256) launch_tree<D, 4>(a, st);
    };
    if (d == 64) go(std::integral_constant<int, 64>{});
    else if (d == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
    return check_launch("attn_tree");
}
