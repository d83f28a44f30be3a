// Verification of drafted tokens against the target's probabilities (include/scmx_cache.h, scmx_verify_drafts).
//
// The residual of a node after k refused children is r_k = max(a_k e - b_k q, 0), e the exponentials of the node's logits, q the
// draft's row, with a_0 = 1 / sum e, b_0 = 0: from r_{k+1} = max(r_k - q, 0) / S and max(max(x, 0) - q, 0) = max(x - q, 0) for q >= 0
// follow S_{k+1} = sum max(a_k e - (b_k + 1) q, 0), a_{k+1} = a_k / S, b_{k+1} = (b_k + 1) / S.  None of it depends on which tokens
// were drafted or taken, so one launch a level forms the sums of all nodes side by side, by chunks of the vocabulary, and the walk
// itself is a single pass over the nodes with scalars.  The chunks' sums then say in which chunk the next token lies, and only
// that chunk is looked at again.  Without a draft q is one-hot: the refused tokens' exponentials leave the sum.  What remains is never
// formed as a difference, which after refusals of nearly all probability would be rounding: the sums leave out the tokens of a
// node's children, and the walk adds those that were not refused.
// Everything is float64 (exponentials too): a sum of 150000 float32 probabilities is uncertain by more than the likelihood of most
// tokens, and which token a random number names has to be the same for every order of summation.
// Bound: float64 arithmetic and one reading of the logits (from the L2 again for each level); a few nodes, the launches.
#include <math.h>

#include <type_traits>

#include "../../include/scmx_cache.h"
#include "scmx_common.h"

namespace scmx {

constexpr int VNT = 256, VCHUNK = 4096, VWALK = 1024, VNODES = 64, VLEVELS = 16;
constexpr int VMAX = VCHUNK * VWALK;   // a thread of the walk per chunk

struct VerifyArgs {
    const int64_t* tokens;
    const int32_t* parents;
    const void* logits;
    const float* draft;
    const float* uniforms;
    int32_t* path;
    int32_t* count;
    int64_t* next;
    int T, V, chunks, levels;
    double rate;       // 64 / (ln 2 temperature)
    bool logits_vec, draft_vec;
    double* z;         // [T][chunks]: sums of a chunk relative to its largest logit, without a draft those of the tokens that no child
                       // of the node holds (greedy: int32, where the largest is)
    double* s;         // [levels][T][chunks]: S_1 ...
    float* m;          // [T][chunks]: largest logits
};

// 2^(j / 64).  The kernels copy it to LDS.
__device__ const double EXP2_64[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0};

// 2^(t / 64), t <= 0, to some 1e-15 (1e-14 at t = -10000): t = k + f, |f| <= 1/2, 2^(f / 64) by the series of exp(f ln 2 / 64) to the fifth
// power (the sixth is 4e-17), 2^(k / 64) from the table and the exponent.  Below 2^-1074: 0.  Half of the time of the stats kernel is
// this arithmetic (60 nodes of 151936: 13.0 us; a series to the eleventh power without a table took 6 more).
__device__ __forceinline__ double exp2_64(double t, const double* table) {
    constexpr double L = 0.010830424696249145;   // ln 2 / 64
    t = fmax(t, -75000.0);
    const double n = rint(t), f = t - n;
    double p = __builtin_fma(f, L * L * L * L * L / 120.0, L * L * L * L / 24.0);
    p = __builtin_fma(p, f, L * L * L / 6.0);
    p = __builtin_fma(p, f, L * L / 2.0);
    p = __builtin_fma(p, f, L);
    p = __builtin_fma(p, f, 1.0);
    const int k = int(n);
    return __builtin_ldexp(p * table[k & 63], k >> 6);
}
// A logit's weight relative to the largest, m: 1 for the largest itself, also where that is infinite.
__device__ __forceinline__ double weight(float x, float m, double rate, const double* table) {
    if (!(fabsf(m) <= 3.4028234e38f)) return x == m ? 1.0 : 0.0;   // (the same for a whole row)
    return exp2_64((double(x) - double(m)) * rate, table);
}
// The same of N logits of which the first `there` are some (the others are -inf): straight code where the largest is finite.
template <int N>
__device__ __forceinline__ void weights(const float* x, float m, double rate, const double* table, int there, double* w) {
    if (fabsf(m) <= 3.4028234e38f) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = exp2_64((double(x[i]) - double(m)) * rate, table);
    } else {
        for (int i = 0; i < N; ++i) w[i] = i < there && x[i] == m ? 1.0 : 0.0;
    }
}
__device__ __forceinline__ void copy_table(double* table) {
    if (threadIdx.x < 64) table[threadIdx.x] = EXP2_64[threadIdx.x];   // (a barrier follows before its first use)
}

__device__ __forceinline__ float clean(float x) { return fmaxf(x, -__builtin_inff()); }   // NaN: -inf
template <bool F32>
__device__ __forceinline__ float logit(const void* logits, size_t at) {
    return clean(F32 ? static_cast<const float*>(logits)[at] : bf16_to_f32(static_cast<const uint16_t*>(logits)[at]));
}
// Eight consecutive logits from token v on (beyond the vocabulary: -inf).
template <bool F32>
__device__ __forceinline__ void logits8(const VerifyArgs& a, size_t row, int v, float* x) {
    if (a.logits_vec && v + 8 <= a.V) {
        if (F32) {
            const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(a.logits) + row * a.V + v);
            const f32x4 lo = p[0], hi = p[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = clean(lo[i]);
                x[4 + i] = clean(hi[i]);
            }
        } else {
            const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.logits) + row * a.V + v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = clean(bf16_lo(w[i]));
                x[2 * i + 1] = clean(bf16_hi(w[i]));
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = v + i < a.V ? logit<F32>(a.logits, row * a.V + v + i) : -__builtin_inff();
}

__device__ __forceinline__ double lane_of(double v, int lane) {
    const long long b = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_readlane(int(b), lane), hi = __builtin_amdgcn_readlane(int(b >> 32), lane);
    return __longlong_as_double((long long)(uint64_t(uint32_t(hi)) << 32 | uint32_t(lo)));
}
template <int CTRL>
__device__ __forceinline__ double row_op(double v) {   // v of the lane that CTRL names; 0 where it names none
    const long long b = __double_as_longlong(v);
    const int lo = __builtin_amdgcn_update_dpp(0, int(b), CTRL, 0xF, 0xF, true);
    const int hi = __builtin_amdgcn_update_dpp(0, int(b >> 32), CTRL, 0xF, 0xF, true);
    return __longlong_as_double((long long)(uint64_t(uint32_t(hi)) << 32 | uint32_t(lo)));
}
// Over the wave, in every lane: within rows of 16 lanes by row operations, the four rows as scalars (a butterfly through LDS has six
// trips of a hundred cycles, and these kernels are chains of such sums).
__device__ __forceinline__ double wave_sum64(double v) {
    v += row_op<0xB1>(v);    // quad_perm 1 0 3 2
    v += row_op<0x4E>(v);    // quad_perm 2 3 0 1
    v += row_op<0x141>(v);   // row_half_mirror
    v += row_op<0x140>(v);   // row_mirror
    return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}
template <int CTRL>
__device__ __forceinline__ float row_max(float v) {
    const int b = __float_as_int(v);
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(b, b, CTRL, 0xF, 0xF, true)));
}
__device__ __forceinline__ float wave_max32(float v) {
    v = row_max<0xB1>(v);
    v = row_max<0x4E>(v);
    v = row_max<0x141>(v);
    v = row_max<0x140>(v);
    const auto at = [&](int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); };
    return fmaxf(fmaxf(at(0), at(16)), fmaxf(at(32), at(48)));
}
// Inclusive sum in lane order.
__device__ __forceinline__ double wave_scan64(double v) {
    v += row_op<0x111>(v);   // row_shr 1, 2, 4, 8
    v += row_op<0x112>(v);
    v += row_op<0x114>(v);
    v += row_op<0x118>(v);
    const double a = lane_of(v, 15), b = lane_of(v, 31), c = lane_of(v, 47);
    const int row = (threadIdx.x & 63) >> 4;
    return v + (row == 0 ? 0.0 : row == 1 ? a : row == 2 ? a + b : (a + b) + c);
}
// What a lane wrote to LDS before is what the wave's other lanes read after.
__device__ __forceinline__ void wave_sees() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// Over the workgroup; every thread gets the result.  `s` holds one entry a wave.
__device__ __forceinline__ float group_max(float v, float* s) {
    v = wave_max32(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
    for (unsigned w = 1; w < blockDim.x / 64; ++w) v = fmaxf(v, s[w]);
    return v;
}
__device__ __forceinline__ double group_sum64(double v, double* s) {
    v = wave_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
    for (unsigned w = 1; w < blockDim.x / 64; ++w) v += s[w];
    return v;
}

// blockIdx.x: chunk, y: node.  A chunk's largest logit and the sum of its weights relative to that (GREEDY: the lowest token that
// holds it).
template <bool F32, bool GREEDY>
__global__ __launch_bounds__(VNT) void verify_stats_kernel(const VerifyArgs a) {
    __shared__ float s_m[VNT / 64];
    __shared__ double s_z[VNT / 64];
    __shared__ int s_at[VNT / 64];
    __shared__ double s_table[64];
    if (!GREEDY) copy_table(s_table);
    const size_t row = blockIdx.y;
    float x[2][8], m = -__builtin_inff();
    const int v0 = blockIdx.x * VCHUNK + 8 * threadIdx.x, lane = threadIdx.x & 63;
    const bool leaves = !GREEDY && !a.draft && lane < a.T;
    const int parent = leaves ? a.parents[lane] : -1;
    const int64_t held = leaves ? a.tokens[lane] - int64_t(blockIdx.x) * VCHUNK : -1;
#pragma unroll
    for (int t = 0; t < 2; ++t) logits8<F32>(a, row, v0 + t * 8 * VNT, x[t]);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, x[t][i]);
    m = group_max(m, s_m);
    const size_t out = row * a.chunks + blockIdx.x;
    if (GREEDY) {
        int at = a.V - 1;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (v0 + t * 8 * VNT + i < a.V && x[t][i] == m) at = min(at, v0 + t * 8 * VNT + i);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) at = min(at, __shfl_xor(at, off, WAVE));
        if ((threadIdx.x & 63) == 0) s_at[threadIdx.x >> 6] = at;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < VNT / 64; ++w) at = min(at, s_at[w]);
            a.m[out] = m;
            reinterpret_cast<int32_t*>(a.z)[out] = at;
        }
        return;
    }
    uint64_t kids = __ballot(parent == int(blockIdx.y) && parent < lane && held >= 0 && held < VCHUNK);   // (the same in every wave)
    while (kids) {
        const int at = __builtin_amdgcn_readlane(int(held), __builtin_ctzll(kids));
        kids &= kids - 1;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (8 * int(threadIdx.x) + t * 8 * VNT + i == at) x[t][i] = __builtin_nanf("");   // weighs 0, whatever m is
    }
    double z = 0.0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        double w[8];
        weights<8>(x[t], m, a.rate, s_table, a.V - (v0 + t * 8 * VNT), w);
#pragma unroll
        for (int i = 0; i < 8; ++i) z += w[i];
    }
    z = group_sum64(z, s_z);
    if (threadIdx.x == 0) {
        a.m[out] = m;
        a.z[out] = z;
    }
}

// a_k, b_k from what came before: one step (S not above zero: nothing is left, the residual stays as it was).
__device__ __forceinline__ void next_level(double s, double& ak, double& bk) {
    if (s > 0.0) {
        ak = ak / s;
        bk = (bk + 1.0) / s;
    }
}

// blockIdx.x: chunk, y: node.  The chunk's part of S_level, for nodes with that many children.
template <bool F32>
__global__ __launch_bounds__(VNT) void verify_level_kernel(const VerifyArgs a, int level) {
    __shared__ float s_m[VNT / 64];
    __shared__ double s_z[VNT / 64], s_table[64];
    copy_table(s_table);
    const int row = blockIdx.y, lane = threadIdx.x & 63;
    if (__popcll(__ballot(lane < a.T && a.parents[min(lane, a.T - 1)] == row)) < level) return;   // (the same in every wave)
    float x[2][8], q[2][8];
    const int v0 = blockIdx.x * VCHUNK + 8 * threadIdx.x;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int v = v0 + t * 8 * VNT;
        logits8<F32>(a, size_t(row), v, x[t]);
        const float* p = a.draft + size_t(row) * a.V + v;
        if (a.draft_vec && v + 8 <= a.V) {
            const f32x4 lo = reinterpret_cast<const f32x4*>(p)[0], hi = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                q[t][i] = lo[i];
                q[t][4 + i] = hi[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[t][i] = v + i < a.V ? p[i] : 0.0f;
        }
    }
    const float* pm = a.m + size_t(row) * a.chunks;
    const double* pz = a.z + size_t(row) * a.chunks;
    float m = -__builtin_inff();
    for (int c = threadIdx.x; c < a.chunks; c += VNT) m = fmaxf(m, pm[c]);
    m = group_max(m, s_m);
    double z = 0.0;
    for (int c = threadIdx.x; c < a.chunks; c += VNT) z += pz[c] * weight(pm[c], m, a.rate, s_table);
    double ak = 1.0 / group_sum64(z, s_z), bk = 0.0;
    for (int l = 1; l < level; ++l) {
        const double* ps = a.s + (size_t(l - 1) * a.T + row) * a.chunks;
        double s = 0.0;
        for (int c = threadIdx.x; c < a.chunks; c += VNT) s += ps[c];
        next_level(group_sum64(s, s_z), ak, bk);
    }
    double s = 0.0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        double w[8];
        weights<8>(x[t], m, a.rate, s_table, a.V - (v0 + t * 8 * VNT), w);
#pragma unroll
        for (int i = 0; i < 8; ++i) s += fmax(ak * w[i] - (bk + 1.0) * double(q[t][i]), 0.0);   // (beyond the vocabulary q is 0)
    }
    s = group_sum64(s, s_z);
    if (threadIdx.x == 0) a.s[(size_t(level - 1) * a.T + row) * a.chunks + blockIdx.x] = s;
}

// Inclusive sum over the workgroup's threads in thread order; `s` holds one entry a wave.
__device__ __forceinline__ double group_scan(double v, double* s) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    v = wave_scan64(v);
    if (lane == 63) s[wave] = v;
    __syncthreads();
    double before = lane < wave ? s[lane] : 0.0;   // (up to 16 waves)
    return v + wave_sum64(before);
}

// One workgroup: the nodes' sums from the chunks', the walk, the token after it.  A chain of trips to memory and of cross-lane
// sums: a wave takes four nodes' sums side by side, and the walk is a wave's, node c's numbers in lane c and read from there as
// scalars (by a thread, over LDS, it took 150 cycles a node: 60 nodes 42 us in all, 8 drawn ones 21).
template <bool F32, bool GREEDY>
__global__ __launch_bounds__(VWALK) void verify_walk_kernel(const VerifyArgs a) {
    constexpr int WAVES = VWALK / 64, PER = VNODES / WAVES;
    __shared__ float s_m[VNODES];
    __shared__ double s_z[VNODES], s_wave[WAVES], s_table[64], s_open_e[VNODES], s_base, s_total;
    __shared__ double s_w[GREEDY ? 1 : VNODES][64];   // the first 64 chunks' sums relative to the node's largest logit
    __shared__ double s_a[GREEDY ? 1 : VNODES][VLEVELS + 1], s_b[GREEDY ? 1 : VNODES][VLEVELS + 1];
    __shared__ int s_best[VNODES], s_level[GREEDY ? 1 : VNODES][VLEVELS + 1], s_last, s_lvl, s_gones, s_chunk, s_over[WAVES], s_some[WAVES];
    __shared__ int s_gone[VNODES], s_open[VNODES], s_again[VNODES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (!GREEDY) copy_table(s_table);
    // node `lane`: every wave knows the parents (it counts children) and tokens, the first one the rest
    const int parent = lane > 0 && lane < a.T ? a.parents[lane] : -1;
    const bool node = lane > 0 && lane < a.T && parent >= 0 && parent < lane;
    const int64_t given = lane < a.T ? a.tokens[lane] : -1;
    const bool known = node && given >= 0 && given < a.V;
    const int token = known ? int(given) : -1 - lane;   // (one that no other node holds)
    float u = 0.0f, x = 0.0f, q = 0.0f;
    if (wave == 0) {
        if (!GREEDY) {
            if (lane < a.T) u = a.uniforms[lane];
            if (known) x = logit<F32>(a.logits, size_t(parent) * a.V + token);
            if (known && a.draft) q = a.draft[size_t(parent) * a.V + token];
        }
    }
    // ---- the sums of nodes wave, wave + 16, ..
    {
        float pm[PER], m[PER];
        double pz[PER], z[PER];
        int at[PER];
#pragma unroll
        for (int r = 0; r < PER; ++r) {
            const int row = min(wave + WAVES * r, a.T - 1);
            const size_t c = size_t(row) * a.chunks + min(lane, a.chunks - 1);
            pm[r] = lane < a.chunks ? a.m[c] : -__builtin_inff();
            if (GREEDY) at[r] = reinterpret_cast<const int32_t*>(a.z)[c];
            else pz[r] = a.z[c];
            m[r] = pm[r];
        }
#pragma unroll 1
        for (int c = 64 + lane; c < a.chunks; c += 64)
#pragma unroll
            for (int r = 0; r < PER; ++r) m[r] = fmaxf(m[r], a.m[size_t(min(wave + WAVES * r, a.T - 1)) * a.chunks + c]);
#pragma unroll
        for (int r = 0; r < PER; ++r) m[r] = wave_max32(m[r]);
        if (GREEDY) {
#pragma unroll
            for (int r = 0; r < PER; ++r) {
                const int row = wave + WAVES * r;
                if (row >= a.T) break;
                int best = lane < a.chunks && pm[r] == m[r] ? at[r] : a.V - 1;
                for (int c = 64 + lane; c < a.chunks; c += 64) {
                    const size_t i = size_t(row) * a.chunks + c;
                    if (a.m[i] == m[r]) best = min(best, reinterpret_cast<const int32_t*>(a.z)[i]);
                }
#pragma unroll
                for (int off = 32; off >= 1; off >>= 1) best = min(best, __shfl_xor(best, off, WAVE));
                if (lane == 0) s_best[row] = best;
            }
        } else {
#pragma unroll
            for (int r = 0; r < PER; ++r) {   // whether an earlier sibling holds the same token
                const int c = wave + WAVES * r, pc = __builtin_amdgcn_readlane(parent, c), tc = __builtin_amdgcn_readlane(token, c);
                const bool again = __ballot(lane < c && parent == pc && token == tc) != 0;
                if (lane == 0) s_again[c] = again;
            }
            __syncthreads();   // the table
#pragma unroll
            for (int r = 0; r < PER; ++r) {
                z[r] = lane < a.chunks ? pz[r] * weight(pm[r], m[r], a.rate, s_table) : 0.0;
                if (wave + WAVES * r < a.T) s_w[wave + WAVES * r][lane] = z[r];
            }
#pragma unroll
            for (int r = 0; r < PER; ++r) z[r] = wave_sum64(z[r]);
#pragma unroll
            for (int r = 0; r < PER; ++r)
                if (lane == 0 && wave + WAVES * r < a.T) {
                    s_m[wave + WAVES * r] = m[r];
                    s_z[wave + WAVES * r] = z[r];
                    s_level[wave + WAVES * r][0] = 0;
                }
        }
    }
    wave_sees();
    if (!GREEDY && a.chunks > 64) {   // the chunks past the lanes
#pragma unroll 1
        for (int row = wave; row < a.T; row += WAVES) {
            double more = 0.0;
#pragma unroll 1
            for (size_t i = size_t(row) * a.chunks + 64 + lane; i < size_t(row + 1) * a.chunks; i += 64)
                more += a.z[i] * weight(a.m[i], s_m[row], a.rate, s_table);
            more = wave_sum64(more);
            if (lane == 0) s_z[row] += more;
        }
        wave_sees();
    }
    if (!GREEDY && a.levels > 0) {
#pragma unroll 1
        for (int row = wave; row < a.T; row += WAVES) {
            double ak = 1.0 / s_z[row], bk = 0.0;   // (this wave's own)
            int level = 0;   // the last one that left something
            if (lane == 0) {
                s_a[row][0] = ak;
                s_b[row][0] = bk;
            }
            const int kids = min(a.levels, int(__popcll(__ballot(node && parent == row))));
#pragma unroll 1
            for (int l = 1; l <= kids; ++l) {
                const double* ps = a.s + (size_t(l - 1) * a.T + row) * a.chunks;
                double s = 0.0;
#pragma unroll 1
                for (int c = lane; c < a.chunks; c += 64) s += ps[c];
                s = wave_sum64(s);
                next_level(s, ak, bk);
                if (s > 0.0) level = l;
                if (lane == 0) {
                    s_a[row][l] = ak;
                    s_b[row][l] = bk;
                    s_level[row][l] = level;
                }
            }
        }
    }
    __syncthreads();
    if (wave == 0) {
        const double e = known && !GREEDY ? weight(x, s_m[max(parent, 0)], a.rate, s_table) : 0.0, qd = known && a.draft ? double(q) : 1.0;
        const bool right = GREEDY && node && token == s_best[max(parent, 0)];
        int cur = 0, tried = 0;
        uint64_t taken = 1, gone = 0;   // gone: children of cur whose tokens were refused
        const bool once = !GREEDY && !a.draft && known && !s_again[lane];
        // what is left of cur's sum: the tokens that no child holds and, each once, those that are not gone
        const auto rest = [&]() { return s_z[cur] + wave_sum64(once && parent == cur && !(gone >> lane & 1) ? e : 0.0); };
        double left = GREEDY || a.draft ? 0.0 : rest();
        uint64_t kids = __ballot(node && parent == 0);
        const uint64_t yes = __ballot(right);
        while (kids) {   // children come after their parents
            const int c = __builtin_ctzll(kids);
            kids &= kids - 1;
            bool take;
            if (GREEDY) {
                take = yes >> c & 1;
            } else if (a.draft) {
                if (tried == a.levels) break;
                const double qc = lane_of(qd, c), r = fmax(s_a[cur][tried] * lane_of(e, c) - s_b[cur][tried] * qc, 0.0);
                take = double(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(u), c))) * qc < r;
                ++tried;
            } else {
                const double ec = gone >> c & 1 ? 0.0 : lane_of(e, c);
                take = double(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(u), c))) * left < ec;
                if (!take && ec > 0.0) {
                    const uint64_t before = gone;
                    gone |= __ballot(parent == cur && token == __builtin_amdgcn_readlane(token, c));
                    const double without = rest();
                    if (without > 0.0) left = without;
                    else gone = before;   // nothing would be left: it stays as it was
                }
            }
            if (take) {
                cur = c;
                taken |= 1ull << c;
                gone = 0;
                tried = 0;
                if (!GREEDY && !a.draft) left = rest();
                kids = __ballot(node && parent == c);
            }
        }
        const int count = int(__popcll(taken));
        const uint64_t below = (1ull << lane) - 1;
        if (taken >> lane & 1) a.path[__popcll(taken & below)] = lane;
        if (lane >= count && lane < a.T) a.path[lane] = -1;
        const uint64_t open = __ballot(once && parent == cur && !(gone >> lane & 1));
        if (gone >> lane & 1) s_gone[__popcll(gone & below)] = token;
        if (open >> lane & 1) {
            s_open[__popcll(open & below)] = token;
            s_open_e[__popcll(open & below)] = e;
        }
        wave_sees();
        if (lane == 0) {
            a.count[0] = count;
            if (GREEDY) a.next[0] = s_best[cur];
        }
        if (!GREEDY) {
            // ---- the chunk that the next token is in: lane i sums chunks i K .. (i + 1) K - 1
            const int lvl = s_level[cur][tried], gones = int(__popcll(gone)), opens = int(__popcll(open)), K = (a.chunks + 63) / 64;
            const auto part = [&](int c) {   // of the residual, in the units of the sums that it was taken from
                if (c >= a.chunks) return 0.0;
                if (lvl > 0) return a.s[(size_t(lvl - 1) * a.T + cur) * a.chunks + c];
                const size_t at = size_t(cur) * a.chunks + c;
                double w = c < 64 ? s_w[cur][c] : a.z[at] * weight(a.m[at], s_m[cur], a.rate, s_table);
                for (int i = 0; i < opens; ++i)
                    if (s_open[i] / VCHUNK == c) w += s_open_e[i];
                return w;
            };
            double own = 0.0;
#pragma unroll 1
            for (int k = 0; k < K; ++k) own += part(lane * K + k);
            const double upto = wave_scan64(own);
            const double total = lane_of(upto, 63);
            const double target = double(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(u), 0))) * total;
            const uint64_t over = __ballot(own > 0.0 && upto > target), some = __ballot(own > 0.0);
            // (no sum above it: the last that has any)
            const int who = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : 0;
            if (lane == who) {
                double run = upto - own, base = run;
                int chunk = lane * K;
#pragma unroll 1
                for (int k = 0; K > 1 && k < K; ++k) {
                    const double w = part(lane * K + k);
                    if (w > 0.0) {
                        chunk = lane * K + k;
                        base = run;
                        if (run + w > target) break;
                    }
                    run += w;
                }
                s_chunk = min(chunk, a.chunks - 1);
                s_base = base;
                s_total = target;
                s_last = cur;
                s_lvl = lvl;
                s_gones = gones;
            }
        }
    }
    if (GREEDY) return;
    __syncthreads();
    // ---- that chunk again, four tokens a thread.  Against a draft its sum may be no more than rounding (of differences): then the first
    // token of the chunks behind it that has any probability, or the last of those before it.
    const int cur = s_last, gones = s_gones, lvl = s_lvl, first = s_chunk;
    const double target = s_total, base = s_base;
    const float m = s_m[cur];
    int chunk = first, token_at = -1;
#pragma unroll 1
    for (int step = 1; token_at < 0 && chunk >= 0;) {   // (the same in every thread)
        double upto[4], r[4], sum = 0.0;
        int some = -1, over = -1;   // the thread's last token that has any probability, its first above the target
        const int v0 = chunk * VCHUNK + 4 * tid;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int v = v0 + i;
            r[i] = 0.0;
            if (v < a.V) {
                const double e = weight(logit<F32>(a.logits, size_t(cur) * a.V + v), m, a.rate, s_table);
                if (lvl > 0) {   // (before its normalisation, as the chunks' sums are)
                    r[i] = fmax(s_a[cur][lvl - 1] * e - (s_b[cur][lvl - 1] + 1.0) * double(a.draft[size_t(cur) * a.V + v]), 0.0);
                } else {
                    r[i] = e;
                    for (int j = 0; j < gones; ++j)
                        if (s_gone[j] == v) r[i] = 0.0;
                }
            }
            sum += r[i];
            upto[i] = sum;
            if (r[i] > 0.0) some = v;
        }
        const double before = base + group_scan(sum, s_wave) - sum;
#pragma unroll
        for (int i = 3; i >= 0; --i)
            if (r[i] > 0.0 && (chunk == first ? before + upto[i] > target : step > 0)) over = v0 + i;
        // lanes and waves hold the chunk in order: the first wave's first lane, or the last's last (atomics on one word took 15 us)
        const uint64_t overs = __ballot(over >= 0), somes = __ballot(some >= 0);
        if (lane == 0) {
            s_over[wave] = overs ? __builtin_amdgcn_readlane(over, __builtin_ctzll(overs)) : -1;
            s_some[wave] = somes ? __builtin_amdgcn_readlane(some, 63 - __builtin_clzll(somes)) : -1;
        }
        __syncthreads();
        const int o = lane < WAVES ? s_over[lane] : -1, h = lane < WAVES ? s_some[lane] : -1;
        const uint64_t any = __ballot(o >= 0), rest = __ballot(h >= 0);
        token_at = any    ? __builtin_amdgcn_readlane(o, __builtin_ctzll(any))
                   : rest ? __builtin_amdgcn_readlane(h, 63 - __builtin_clzll(rest))
                          : -1;
        chunk += step;
        if (chunk == a.chunks) {
            step = -1;
            chunk = first - 1;
        }
    }
    if (tid == 0) a.next[0] = max(token_at, 0);
}

}  // namespace scmx

using namespace scmx;

static int verify_chunks(int V) { return int((int64_t(V) + VCHUNK - 1) / VCHUNK); }

extern "C" size_t scmx_verify_workspace(int T, int V, int siblings) {
    if (T < 1 || T > VNODES || V < 1 || V > VMAX || siblings < 0 || siblings > VLEVELS) return 0;
    return size_t(T) * verify_chunks(V) * (sizeof(double) * (1 + siblings) + sizeof(float));
}

extern "C" int scmx_verify_drafts(const int64_t* tokens, const int32_t* parents, const void* logits, int logits_f32, const float* draft,
                                  double temperature, const float* uniforms, int32_t* path, int32_t* count, int64_t* next, int T, int V,
                                  int siblings, void* workspace, size_t workspace_bytes, void* stream) {
    const bool greedy = temperature == 0.0;
    if (!tokens || !parents || !logits || !path || !count || !next || (!greedy && !uniforms)) {
        set_error("verify_drafts: null pointer argument");
        return SCMX_ERR_ARG;
    }
    if (T < 1 || T > VNODES || V < 1 || V > VMAX) {
        set_error("verify_drafts: need 1..%d nodes and a vocabulary of 1..%d (T=%d V=%d)", VNODES, VMAX, T, V);
        return SCMX_ERR_ARG;
    }
    if (!(temperature >= 0.0 && temperature <= 1.0e30) || (!greedy && temperature < 1.0e-6)) {
        set_error("verify_drafts: temperature must be 0 or 1e-6 ... 1e30");
        return SCMX_ERR_ARG;
    }
    if (draft && !greedy && (siblings < 1 || siblings > VLEVELS)) {
        set_error("verify_drafts: a draft needs siblings 1..%d (%d)", VLEVELS, siblings);
        return SCMX_ERR_ARG;
    }
    const int levels = draft && !greedy ? siblings : 0, chunks = verify_chunks(V);
    const size_t need = scmx_verify_workspace(T, V, levels);
    if (!workspace || workspace_bytes < need || uintptr_t(workspace) % 8) {
        set_error("verify_drafts: needs %zu bytes of workspace, 8-byte aligned", need);
        return SCMX_ERR_WORKSPACE;
    }
    const size_t cells = size_t(T) * chunks;
    VerifyArgs a{tokens, parents, logits, greedy ? nullptr : draft, uniforms, path, count, next, T, V, chunks, levels,
                 greedy ? 1.0 : 64.0 / M_LN2 / temperature,
                 uintptr_t(logits) % 16 == 0 && V % (logits_f32 ? 4 : 8) == 0, uintptr_t(draft) % 16 == 0 && V % 4 == 0,
                 static_cast<double*>(workspace), static_cast<double*>(workspace) + cells, nullptr};
    a.m = reinterpret_cast<float*>(a.s + cells * levels);
    const hipStream_t st = (hipStream_t)stream;
    const dim3 grid(chunks, T);
    const auto go = [&](auto f32) {
        constexpr bool F32 = decltype(f32)::value;
        if (greedy) {
            verify_stats_kernel<F32, true><<<grid, dim3(VNT), 0, st>>>(a);
            verify_walk_kernel<F32, true><<<dim3(1), dim3(VWALK), 0, st>>>(a);
            return;
        }
        verify_stats_kernel<F32, false><<<grid, dim3(VNT), 0, st>>>(a);
        for (int l = 1; l <= levels; ++l) verify_level_kernel<F32><<<grid, dim3(VNT), 0, st>>>(a, l);
        verify_walk_kernel<F32, false><<<dim3(1), dim3(VWALK), 0, st>>>(a);
    };
    if (logits_f32) go(std::true_type{});
    else go(std::false_type{});
    return check_launch("verify_drafts");
}
