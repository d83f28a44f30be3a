// Attention of a tree of drafted tokens (1..64 of them, one: a decode step) against a KV cache in 4 bits (include/scmx_mx.h,
// scmx_attn_tree4).
//
// As over bf16 and 8-bit caches (attn_tree.hip): the query heads of a KV head and their tokens are the rows of one matrix product, a wave
// owns 16 or 32 of them and walks tiles of 32 keys with a running reference, both products are transposed so that a query is a lane
// column in both and the scores' accumulators are the second product's operand where they are, and nothing is staged.
//
// S^T = K Q^T runs on the scaled matrix instruction 16x16x128, the K codes and their bytes as they lie in the cache: no conversion.  The
// queries are its other operand in E4M3, as two parts: hi, rounded to four bits, with the block's exponent, and lo, what is left (exact
// in four bits more: q has eight), with an exponent 5 lower.  Both are exact for values down to 2^-14 of the block's largest, below that
// their sum is off by at most 2^-23 of it.  64 dimensions take both parts in one instruction (K twice), 128 an instruction each, 256 two.
// The instruction's E2M1 operand is 32 consecutive values a lane (lane group g: 32 g ..), its E4M3 operand 16 g .. and 64 + 16 g ..; a
// byte belongs to the 32 values from 32 g on in both.
// O^T = V^T P^T in bf16: a lane reads DPL = d / 16 consecutive codes of eight V rows, the conversion applies the row's block scale (exact
// in bf16), byte permutes pair the rows.  The weights are two bf16 parts, what rounds to bf16 and what is left, 16 bits in all, and each
// product is two: in one part (2^-8) the weights' rounding was as large as the result's, and larger where values cancel.  One token over
// 300 / 40000 rows of 16:8 x 128 6.3 / 13.1 us, 64 tokens over 6000 of 32:8 x 128 20.6 (in one part 6.0 / 12.6 / 18.6).
#include <math.h>

#include <type_traits>
#include <utility>

#include "attn_tree.h"
#include "mx.h"

namespace scmx {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short i16x2 __attribute__((ext_vector_type(2)));

struct Tree4Args : TreeArgs {
    const uint8_t* ksb;
    const uint8_t* vsb;
};

constexpr int FP4 = 4, FP8 = 0;   // of the instruction's format operands
constexpr uint32_t LO_STEP = 5;   // powers of two from a block's exponent to that of what is left

template <typename F, int... E>
__device__ __forceinline__ void for_each(F&& f, std::integer_sequence<int, E...>) { (f(std::integral_constant<int, E>{}), ...); }

// 16 bf16 values (a lane's half of a block of 32, the other half 16 lanes away) as E4M3 codes hi and lo; returns the block's byte.
__device__ __forceinline__ uint32_t split_e4m3(const u32x4 (&q)[2], uint32_t (&hi)[4], uint32_t (&lo)[4]) {
    uint32_t top = 0;
    float x[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[2 * i] = bf16_lo(q[i / 4][i % 4]);
        x[2 * i + 1] = bf16_hi(q[i / 4][i % 4]);
        top = max(top, max(__float_as_uint(x[2 * i]) & 0x7FFFFFFFu, __float_as_uint(x[2 * i + 1]) & 0x7FFFFFFFu));
    }
    top = max(top, uint32_t(__shfl_xor(int(top), 16, WAVE)));
    // the largest value in 2^7 .. 2^8 (448 is E4M3's largest); an infinity or NaN becomes NaN
    const uint32_t e = top >> 23, byte = e == 255 ? 255 : e < 7 + LO_STEP ? LO_STEP : e - 7;
    const float s = mx_scale(byte), sl = mx_scale(byte - LO_STEP);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        i16x2 h = {0, 0}, l = {0, 0};
        h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, x[4 * i], x[4 * i + 1], s, false);
        h = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(h, x[4 * i + 2], x[4 * i + 3], s, true);
        hi[i] = __builtin_bit_cast(uint32_t, h);
        const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi[i], s, false);
        const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi[i], s, true);
        l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, x[4 * i] - a[0], x[4 * i + 1] - a[1], sl, false);
        l = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(l, x[4 * i + 2] - b[0], x[4 * i + 3] - b[1], sl, true);
        lo[i] = __builtin_bit_cast(uint32_t, l);
    }
    return byte;
}

template <int D, int RT>
__global__ __launch_bounds__(TNT, 2) void attn_tree4_kernel(const Tree4Args a) {
    constexpr int ROWB = D / 2, NB = D / 32;       // bytes of codes and of scales of a cache row
    constexpr int KL = D == 256 ? 2 : 1;           // 16-byte loads of a lane from a K row
    constexpr int QN = D == 64 ? 1 : 2 * KL;       // instructions a score tile: operands of a query
    constexpr int DPL = D / 16;                    // head-dimension indexes of a lane in V^T, and MFMAs of the second product
    constexpr int VW = D == 256 ? 2 : 1;           // words of a lane from a V row (d 64: half of one)
    constexpr int ROWS = 16 * RT, WAVES = TWAVES, NT = TNT;
    constexpr float NEG = -__builtin_inff();
    constexpr float PASS = 8.0f;   // how far scores may pass the reference, in powers of two
    __shared__ float s_o[WAVES][ROWS][D + 4];
    __shared__ float s_m[WAVES][ROWS], s_l[WAVES][ROWS];   // references, denominators

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
    const uint8_t* ksb = a.ksb + size_t(kvh) * a.rows * NB;
    const uint8_t* vsb = a.vsb + size_t(kvh) * a.rows * NB;
    u32x4 kr[2][KL];
    uint32_t ks[2][KL];    // the byte of the lane's block
    uint32_t vr[8][VW];
    uint32_t vs[VW];       // all bytes of one row: lane j of eight holds the row of the lane's key j
    const int kg = D == 64 ? g % 2 : g;   // the block of a K row that the lane holds (256: and the one four later)
    const auto load_k = [&](int tile) __attribute__((always_inline)) {
        const int base = tile * TKEYS;
        const auto row = [&](int i) { return min(i, n - 1 - base); };
        const uint8_t *kt = kb + size_t(base) * ROWB, *st = ksb + size_t(base) * NB;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int u = 0; u < KL; ++u) {
                kr[h][u] = *reinterpret_cast<const u32x4*>(kt + unsigned(row(16 * h + ln) * ROWB + 16 * (kg + 4 * u)));
                ks[h][u] = st[unsigned(row(16 * h + ln) * NB + kg + 4 * u)];
            }
    };
    const auto load_v = [&](int tile) __attribute__((always_inline)) {
        const int base = tile * TKEYS;
        const auto row = [&](int i) { return min(i, n - 1 - base); };
        const uint8_t *vt = vb + size_t(base) * ROWB, *st = vsb + size_t(base) * NB;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint8_t* p = vt + unsigned(row(16 * (e / 4) + 4 * g + e % 4) * ROWB + ROWB / 16 * ln);
            if constexpr (D == 64) {
                vr[e][0] = *reinterpret_cast<const uint16_t*>(p);
            } else if constexpr (D == 128) {
                vr[e][0] = *reinterpret_cast<const uint32_t*>(p);
            } else {
                const u32x2 w = *reinterpret_cast<const u32x2*>(p);
                vr[e][0] = w[0];
                vr[e][1] = w[1];
            }
        }
        const uint8_t* p = st + unsigned(row(16 * (ln / 4 % 2) + 4 * g + ln % 4) * NB);
        if constexpr (D == 64) {
            vs[0] = *reinterpret_cast<const uint16_t*>(p);
        } else if constexpr (D == 128) {
            vs[0] = *reinterpret_cast<const uint32_t*>(p);
        } else {
            const u32x2 w = *reinterpret_cast<const u32x2*>(p);
            vs[0] = w[0];
            vs[1] = w[1];
        }
    };
    // ---- the queries, in two parts
    i32x8 qf[RT][QN];
    int qs[RT][QN];
    uint64_t seen[RT];
    const int start = first + wave < last ? first + wave : last - 1;   // (a wave without a tile loads one and uses none)
    constexpr int PARTS = D / 64;   // pieces of 64 dimensions, 16 a lane
    u32x4 qraw[RT][PARTS][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = min(row0 + 16 * rt + ln, rows_all - 1), i = token(r);
        seen[rt] = (a.mask ? uint64_t(a.mask[i]) : ~0ull >> (63 - i)) & ~0ull >> (64 - a.T);
        const uint16_t* qp = a.q + out_row(r) * D + 16 * g;
#pragma unroll
        for (int p = 0; p < PARTS; ++p)
#pragma unroll
            for (int h = 0; h < 2; ++h) qraw[rt][p][h] = *reinterpret_cast<const u32x4*>(qp + 64 * p + 8 * h);
    }
    __builtin_amdgcn_sched_barrier(0);
    load_k(start);
    load_v(start);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        uint32_t hi[PARTS][4], lo[PARTS][4], byte[PARTS];
#pragma unroll
        for (int p = 0; p < PARTS; ++p) byte[p] = split_e4m3(qraw[rt][p], hi[p], lo[p]);
        // a piece has two blocks, whose bytes lie in lane groups 0, 1 and 2, 3; group g needs that of block g
        const int from = 32 * (g % 2) + ln;
        if constexpr (D == 64) {
            const uint32_t b = uint32_t(__shfl(int(byte[0]), from, WAVE));
            qs[rt][0] = int(g < 2 || b == 255 ? b : b - LO_STEP);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                qf[rt][0][w] = int(hi[0][w]);
                qf[rt][0][4 + w] = int(lo[0][w]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < KL; ++u) {
                const uint32_t b0 = uint32_t(__shfl(int(byte[2 * u]), from, WAVE)), b1 = uint32_t(__shfl(int(byte[2 * u + 1]), from, WAVE));
                const uint32_t b = g < 2 ? b0 : b1;
                qs[rt][2 * u] = int(b);
                qs[rt][2 * u + 1] = int(b == 255 ? b : b - LO_STEP);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    qf[rt][2 * u][w] = int(hi[2 * u][w]);
                    qf[rt][2 * u][4 + w] = int(hi[2 * u + 1][w]);
                    qf[rt][2 * u + 1][w] = int(lo[2 * u][w]);
                    qf[rt][2 * u + 1][4 + w] = int(lo[2 * u + 1][w]);
                }
            }
        }
    }
    // Sums of weights up to 2^8 times values up to 6 * 2^125 pass float32.  Of fewer than 2^room rows they do not while a weight times a
    // value's scale is below 2^(122 - room); a query that meets more has its reference 2^(10 + room) higher (lift), until its scores pass
    // even that.  (Not before: weights below 2^(room - 116) are lost then, which count where no other row's product is large.)
    const int room = 32 - __builtin_clz(unsigned(n));
    f32x4 o[RT][DPL], ones[RT];   // ones: sums of the rounded weights
    float m[RT], lift[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        lift[rt] = 0.0f;
#pragma unroll
        for (int i = 0; i < DPL; ++i) o[rt][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        ones[rt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m[rt] = NEG;
    }

    // K of the next tile is requested when this one's scores stand, V when its product does.
    for (int tile = first + wave; tile < last; tile += WAVES) {
        const int base = tile * TKEYS, next = min(tile + WAVES, last - 1);
        const bool tail = base > pos - TKEYS;   // the tile reaches into the tree, or past the last row
        // ---- scores
        f32x4 s[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][0] = s[rt][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int qn = 0; qn < QN; ++qn)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u32x4 c = kr[h][qn / 2];
                const i32x8 kf = {int(c[0]), int(c[1]), int(c[2]), int(c[3]), 0, 0, 0, 0};
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    s[rt][h] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(kf, qf[rt][qn], s[rt][h], FP4, FP8, 0,
                                                                                 int(ks[h][qn / 2]), 0, qs[rt][qn]);
            }
        __builtin_amdgcn_sched_barrier(0);
        load_k(next);
        __builtin_amdgcn_sched_barrier(0);
        // ---- in powers of two; masked
        float x[RT][8];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[rt][e] = s[rt][e / 4][e % 4] * a.scale;
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
            any |= top[rt] > m[rt] + (PASS - lift[rt]);
        }
        if (__builtin_amdgcn_ballot_w64(any)) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float t0 = fmaxf(top[rt], __shfl_xor(top[rt], 16, WAVE));
                t0 = fmaxf(t0, __shfl_xor(t0, 32, WAVE));
                // (each query by its own scores alone: no other query's change what it gets)
                const bool passes = t0 > m[rt] + (PASS - lift[rt]);
                if (t0 >= m[rt]) lift[rt] = 0.0f;   // (what was large is small now)
                const float mn = passes ? t0 + lift[rt] : m[rt];
                const float alpha = mn == NEG ? 1.0f : __builtin_amdgcn_exp2f(m[rt] - mn);
                m[rt] = mn;
#pragma unroll
                for (int r = 0; r < 4; ++r) ones[rt][r] *= alpha;
#pragma unroll
                for (int i = 0; i < DPL; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[rt][i][r] *= alpha;
            }
        }
        // ---- weights
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float shift = m[rt] == NEG ? 0.0f : m[rt];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[rt][e] = __builtin_amdgcn_exp2f(x[rt][e] - shift);
        }
        // ---- scales of the lane's eight keys: its block's byte of each row
        float sv[8];
        for_each([&](auto ec) __attribute__((always_inline)) {
            constexpr int E = decltype(ec)::value;
            uint32_t w = dpp<ROW_SHARE + E>(vs[0]);
            if constexpr (D == 256) {
                const uint32_t other = dpp<ROW_SHARE + E>(vs[1]);   // (by all lanes: it reads those that take the first)
                w = ln < 8 ? w : other;
            }
            sv[E] = mx_scale(w >> (8 * (ln * DPL / 32 % 4)) & 0xFFu);
        }, std::make_integer_sequence<int, 8>{});
        // ---- large values, from 2^65 on: the two upper bits of a byte
        uint32_t large = vs[0] & vs[0] << 1;
        if constexpr (D == 256) large |= vs[1] & vs[1] << 1;
        if (__builtin_amdgcn_ballot_w64((large & 0x80808080u) != 0)) {
            uint32_t top = 0;   // the largest byte of the row that the lane holds (a NaN's is none)
#pragma unroll
            for (int i = 0; i < 4 * VW; ++i) {
                const uint32_t byte = vs[i / 4] >> (8 * (i % 4)) & 0xFFu;
                top = byte == 255 ? top : max(top, byte);
            }
            float most[8];   // the largest scale of the lane's keys
            for_each([&](auto ec) __attribute__((always_inline)) {
                constexpr int E = decltype(ec)::value;
                most[E] = mx_scale(dpp<ROW_SHARE + E>(top));
            }, std::make_integer_sequence<int, 8>{});
            const float least = mx_scale(uint32_t(127 + 122 - room));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                bool meets = false;
#pragma unroll
                for (int e = 0; e < 8; ++e) meets |= x[rt][e] * most[e] >= least;
                const uint64_t b = __builtin_amdgcn_ballot_w64(meets && lift[rt] == 0.0f);
                const uint64_t column = b | b >> 32;   // of the query's four lanes any
                if (!((column | column >> 16) >> ln & 1)) continue;
                lift[rt] = float(10 + room);
                const float higher = m[rt] + lift[rt], down = __builtin_amdgcn_exp2f(m[rt] - higher);   // (m is finite: it has weights)
                m[rt] = higher;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[rt][e] *= down;
#pragma unroll
                for (int r = 0; r < 4; ++r) ones[rt][r] *= down;
#pragma unroll
                for (int i = 0; i < DPL; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[rt][i][r] *= down;
            }
        }
        u32x4 pf[RT], pl[RT];   // the weights to bf16, and what that leaves off
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                pf[rt][e] = f32_to_bf16x2(x[rt][2 * e], x[rt][2 * e + 1]);
                pl[rt][e] = f32_to_bf16x2(x[rt][2 * e] - bf16_lo(pf[rt][e]), x[rt][2 * e + 1] - bf16_hi(pf[rt][e]));
            }
        // ---- the tree's rows: a NaN must not reach (0 times NaN) the queries that do not see its row
        if (tail) {
            uint32_t bad = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int key = base + 16 * (e / 4) + 4 * g + e % 4;
                const bool nan = key >= pos && __float_as_uint(sv[e]) == 0x7F800000u;
                const uint64_t b = __builtin_amdgcn_ballot_w64(nan);
                const uint32_t of = uint32_t((b & 0xFFFFu) != 0) | uint32_t((b >> 16 & 0xFFFFu) != 0) << 1 |
                                    uint32_t((b >> 32 & 0xFFFFu) != 0) << 2 | uint32_t((b >> 48) != 0) << 3;
                bad |= of << (4 * e);
                if (nan) sv[e] = 1.0f;
            }
            for (; bad; bad &= bad - 1) {   // rare: NaN by hand to those that see the row
                const int at = __builtin_ctz(bad), key = base + 16 * (at / 16) + 4 * (at % 4) + at / 4 % 4;
                if (key >= n) continue;   // (behind the last row: a copy of that)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint8_t byte = vsb[size_t(key) * NB + DPL * (4 * g + r) / 32];
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        if (byte == 255 && (seen[rt] >> (key - pos) & 1)) {
#pragma unroll
                            for (int i = 0; i < DPL; ++i) o[rt][i][r] = __builtin_nanf("");
                        }
                }
            }
        }
        // ---- O^T += V^T P^T
        const u32x4 one = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
        const auto multiply = [](u32x4 v, u32x4 p, f32x4 sum) __attribute__((always_inline)) {
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v), __builtin_bit_cast(bf16x8, p), sum, 0, 0, 0);
        };
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) ones[rt] = multiply(one, pl[rt], multiply(one, pf[rt], ones[rt]));
        for_each([&](auto bc) __attribute__((always_inline)) {   // bytes of codes: two head-dimension indexes each
            constexpr int B = decltype(bc)::value;
            u32x4 w0, w1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t lo = mx_bf16x2<B % 4>(vr[2 * e][B / 4], sv[2 * e]);
                const uint32_t hi = mx_bf16x2<B % 4>(vr[2 * e + 1][B / 4], sv[2 * e + 1]);
                w0[e] = perm(hi, lo, 0x05040100u);
                w1[e] = perm(hi, lo, 0x07060302u);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                o[rt][2 * B] = multiply(w0, pf[rt], o[rt][2 * B]);
                o[rt][2 * B + 1] = multiply(w1, pf[rt], o[rt][2 * B + 1]);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                o[rt][2 * B] = multiply(w0, pl[rt], o[rt][2 * B]);
                o[rt][2 * B + 1] = multiply(w1, pl[rt], o[rt][2 * B + 1]);
            }
        }, std::make_integer_sequence<int, DPL / 2>{});
        __builtin_amdgcn_sched_barrier(0);
        load_v(next);
        __builtin_amdgcn_sched_barrier(0);
    }

    // ---- the waves meet: their references first, so that what they leave in LDS only has to be added
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
        if (g == 0) {
            s_m[wave][16 * rt + ln] = m[rt];
            s_l[wave][16 * rt + ln] = ones[rt][0];
        }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = 16 * rt + ln;
        float mw[WAVES], lw[WAVES], mx = NEG, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            mw[w] = s_m[w][r];
            lw[w] = s_l[w][r];
            mx = fmaxf(mx, mw[w]);
        }
#pragma unroll
        for (int w = 0; w < WAVES; ++w)   // (0 of a wave whose keys the query does not see)
            if (lw[w] != 0.0f) sum = __builtin_fmaf(__builtin_amdgcn_exp2f(mw[w] - mx), lw[w], sum);
        float f = ones[rt][0] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(m[rt] - mx);
        if (whole) f *= sum == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(sum);   // (0: nothing was seen)
        else if (wave == 0 && g == 0 && row0 + r < rows_all)
            *reinterpret_cast<float2*>(a.part + size_t(a.T) * a.hq * a.splits * D + 2 * (out_row(row0 + r) * a.splits + range)) =
                float2{mx, sum};
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
static void launch_tree4(const Tree4Args& a, hipStream_t st) {
    const unsigned combos = unsigned(a.hk) * a.splits, grid = (combos + TXCDS - 1) / TXCDS * TXCDS * a.blocks;
    attn_tree4_kernel<D, RT><<<dim3(grid), dim3(TNT), 0, st>>>(a);
    launch_join<D>(a, st);
}

}  // namespace scmx

using namespace scmx;

// 16-row blocks of queries a wave: two where there are that many rows and its registers hold them.
static int tree4_blocks(int qrows, int d) { return qrows <= 16 || d == 256 ? 1 : 2; }

extern "C" int scmx_attn_tree4_splits(int T, int n, int hq, int hk, int d) {
    if (T < 1 || T > 64 || n < 1 || hq < 1 || hk < 1 || hq > 65535 || hq % hk || (d != 64 && d != 128 && d != 256)) return 1;
    const int qrows = T * (hq / hk), rt = tree4_blocks(qrows, d), tiles = tiles_of(n);
    if (tiles <= TONE) return 1;
    // A workgroup a CU, a tile a wave; up to 32 ranges of one tile a wave are 16 of two instead, whose join reads half as much.  Two
    // workgroups a CU where a wave has eight tiles and more.  us in a graph: one token of 16:8 x 128, 16 / 32 / 64 ranges, 3000 rows 7.9 /
    // 8.2 / -, 10000 9.7 / 8.9 / 9.3, 40000 23.2 / 16.1 / 13.8; 64 tokens of 32:8 x 128, 6000 rows, 4 / 8 / 16 ranges 21.4 / 21.6 / 32.0.
    // Eight waves a workgroup (with weights in one part, where four took a few per cent less than now): 40000 rows 14.4 with 32 ranges,
    // 15.2 with 64, 16 tokens of 3000 rows 12.1 (four 10.8), one range of 300 rows 5.9 (6.1), of 500 6.9 (6.6).
    const int64_t groups = int64_t(hk) * ((qrows + 16 * rt - 1) / (16 * rt)), one = 256 / groups;
    const int64_t most = tiles >= 8 * TWAVES * one ? 512 / groups : one;
    const int even = (tiles + TWAVES - 1) / TWAVES, ranges = even > 16 && even <= 32 ? 16 : even < 64 ? even : 64;
    return most < 1 ? 1 : ranges < most ? ranges : int(most);
}

extern "C" int scmx_attn_tree4(const uint16_t* q, const uint8_t* kcache, const uint8_t* vcache, const uint8_t* kscale,
                               const uint8_t* vscale, const int64_t* mask, const int64_t* pos_dev, int64_t pos0, uint16_t* out, int T,
                               int hq, int hk, int d, int cache_rows, float scale, float* workspace, int splits, void* stream) {
    if (!q || !kcache || !vcache || !out || !kscale || !vscale) {
        set_error("attn_tree4: null pointer argument");
        return SCMX_ERR_ARG;
    }
    if (T < 1 || T > 64 || hq < 1 || hk < 1 || hq > 65535 || hq % hk || hq / hk > 4096 || cache_rows < T) {
        set_error("attn_tree4: need 1..64 nodes, hq %% hk == 0, up to 4096 query heads a KV head and a cache that holds the tree "
                  "(T=%d hq=%d hk=%d rows=%d)", T, hq, hk, cache_rows);
        return SCMX_ERR_ARG;
    }
    if (d != 64 && d != 128 && d != 256) {
        set_error("attn_tree4: head dim must be 64, 128 or 256 (d=%d)", d);
        return SCMX_ERR_ARG;
    }
    if (!pos_dev && (pos0 < 0 || pos0 > int64_t(cache_rows) - T)) {
        set_error("attn_tree4: %d rows from %lld on do not fit a cache of %d rows", T, (long long)pos0, cache_rows);
        return SCMX_ERR_ARG;
    }
    if (!(fabsf(scale * 1.4426950408889634f) <= 3.4028234e38f)) {   // (the kernel works in powers of two)
        set_error("attn_tree4: scale must be finite, times log2 e too");
        return SCMX_ERR_ARG;
    }
    if ((uintptr_t(q) | uintptr_t(kcache) | uintptr_t(vcache) | uintptr_t(out)) % 16 ||
        (uintptr_t(kscale) | uintptr_t(vscale)) % (d / 32)) {
        set_error("attn_tree4: q, out and the caches must be 16-byte aligned, scales to a row's bytes");
        return SCMX_ERR_ARG;
    }
    if (splits < 1 || splits > 64 || (splits > 1 && (!workspace || uintptr_t(workspace) % 16))) {
        set_error("attn_tree4: splits must be 1..64 and need a 16-byte aligned workspace of splits * T * hq * (d + 2) floats");
        return SCMX_ERR_ARG;
    }
    const int qrows = T * (hq / hk), rt = tree4_blocks(qrows, d);
    const uint32_t by_group = uint32_t(((uint64_t(1) << 32) + hq / hk - 1) / uint64_t(hq / hk));
    Tree4Args a;
    static_cast<TreeArgs&>(a) = TreeArgs{q, kcache, vcache, nullptr, nullptr, mask, pos_dev, pos0, out, workspace, T, hq, hk, cache_rows,
                                         splits, (qrows + 16 * rt - 1) / (16 * rt), by_group, scale * 1.4426950408889634f};
    a.ksb = kscale;
    a.vsb = vscale;
    const hipStream_t st = (hipStream_t)stream;
    const auto go = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        if (rt == 1) launch_tree4<D, 1>(a, st);
        else if constexpr (D < 256) launch_tree4<D, 2>(a, st);
    };
    if (d == 64) go(std::integral_constant<int, 64>{});
    else if (d == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
    return check_launch("attn_tree4");
}
