// Verification of drafted tokens against the target's probabilities (include/scmx_cache.h, scmx_verify_drafts).
//
// The residual of a node after k refused children is r_k = max(a_k e - b_k q, 0), e the exponentials of the node's logits, q the
// draft's row, with a_0 = 1 / sum e, b_0 = 0: from r_{k+1} = max(r_k - q, 0) / S and max(max(x, 0) - q, 0) = max(x - q, 0) for q >= 0
// follow S_{k+1} = sum max(a_k e - (b_k + 1) q, 0), a_{k+1} = a_k / S, b_{k+1} = (b_k + 1) / S.  None of it depends on which tokens
// were drafted or taken, so one launch a level forms the sums of all nodes side by side, by chunks of the vocabulary, and the walk
// itself is a single pass over the nodes with scalars.  The chunks' sums then say in which chunk the next token lies, and only
// that chunk is looked at again.  Without a draft q is one-hot: the refused tokens' exponentials leave the sum.
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
    double inv_t;      // 1 / temperature
    bool logits_vec, draft_vec;
    double* z;         // [T][chunks]: sums of a chunk relative to its largest logit (greedy: int32, where that is)
    double* s;         // [levels][T][chunks]: S_1 ...
    float* m;          // [T][chunks]: largest logits
};

// exp(x), x <= 0, to some 1e-14: 2^n times the series of what is left, |r| <= ln 2 / 2 (r^12 / 12! = 6e-15).
__device__ __forceinline__ double exp_neg(double x) {
    const double n = rint(fmax(x, -700.0) * 1.4426950408889634);
    double r = __builtin_fma(n, -0.693147180559945286, fmax(x, -700.0));
    r = __builtin_fma(n, -2.319046813846299558e-17, r);
    double p = 1.0 / 39916800.0;
    constexpr double c[] = {1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0, 1.0 / 120.0, 1.0 / 24.0, 1.0 / 6.0, 0.5, 1.0, 1.0};
#pragma unroll
    for (int i = 0; i < 11; ++i) p = __builtin_fma(p, r, c[i]);
    const double v = p * __longlong_as_double((long long)(int(n) + 1023) << 52);
    return x < -700.0 ? 0.0 : v;
}
// A logit's weight relative to the largest, m: 1 for the largest itself, also where it is infinite.
__device__ __forceinline__ double weight(float x, float m, double inv_t) { return x == m ? 1.0 : exp_neg((double(x) - double(m)) * inv_t); }

__device__ __forceinline__ float clean(float x) { return x == x ? x : -__builtin_inff(); }
template <bool F32>
__device__ __forceinline__ float logit(const void* logits, size_t at) {
    return clean(F32 ? static_cast<const float*>(logits)[at] : bf16_to_f32(static_cast<const uint16_t*>(logits)[at]));
}
// Eight consecutive logits from token v on (beyond the vocabulary: anything).
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
    for (int i = 0; i < 8; ++i) x[i] = v + i < a.V ? logit<F32>(a.logits, row * a.V + v + i) : 0.0f;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, WAVE);
    return v;
}
// Over the workgroup; every thread gets the result.  `s` holds one entry a wave.
__device__ __forceinline__ float group_max(float v, float* s) {
    v = wave_max(v);
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
    const size_t row = blockIdx.y;
    float x[2][8], m = -__builtin_inff();
    const int v0 = blockIdx.x * VCHUNK + 8 * threadIdx.x;
#pragma unroll
    for (int t = 0; t < 2; ++t) logits8<F32>(a, row, v0 + t * 8 * VNT, x[t]);
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (v0 + t * 8 * VNT + i < a.V) m = fmaxf(m, x[t][i]);
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
    double z = 0.0;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (v0 + t * 8 * VNT + i < a.V) z += weight(x[t][i], m, a.inv_t);
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
    __shared__ double s_z[VNT / 64];
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
    for (int c = threadIdx.x; c < a.chunks; c += VNT) z += pz[c] * weight(pm[c], m, a.inv_t);
    double ak = 1.0 / group_sum64(z, s_z), bk = 0.0;
    for (int l = 1; l < level; ++l) {
        const double* ps = a.s + (size_t(l - 1) * a.T + row) * a.chunks;
        double s = 0.0;
        for (int c = threadIdx.x; c < a.chunks; c += VNT) s += ps[c];
        next_level(group_sum64(s, s_z), ak, bk);
    }
    double s = 0.0;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (v0 + t * 8 * VNT + i < a.V) s += fmax(ak * weight(x[t][i], m, a.inv_t) - (bk + 1.0) * double(q[t][i]), 0.0);
    s = group_sum64(s, s_z);
    if (threadIdx.x == 0) a.s[(size_t(level - 1) * a.T + row) * a.chunks + blockIdx.x] = s;
}

// Inclusive sum over the workgroup's threads in thread order; `s` holds one entry a wave.
__device__ __forceinline__ double group_scan(double v, double* s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const double up = __shfl_up(v, off, WAVE);
        if (lane >= off) v += up;
    }
    __syncthreads();
    if (lane == 63) s[wave] = v;
    __syncthreads();
    for (int w = 0; w < wave; ++w) v += s[w];
    return v;
}

// One workgroup: the nodes' sums from the chunks', the walk (a thread, over scalars in LDS), the token after it.
template <bool F32, bool GREEDY>
__global__ __launch_bounds__(VWALK) void verify_walk_kernel(const VerifyArgs a) {
    __shared__ float s_m[VNODES];
    __shared__ double s_z[VNODES], s_e[VNODES], s_q[VNODES], s_wave[VWALK / 64];
    __shared__ double s_a[GREEDY ? 1 : VNODES][VLEVELS + 1], s_b[GREEDY ? 1 : VNODES][VLEVELS + 1];
    __shared__ int s_best[VNODES], s_parent[VNODES], s_level[VNODES][VLEVELS + 1], s_gone[VNODES], s_last, s_lvl, s_ngone, s_lo, s_hi;
    __shared__ int64_t s_token[VNODES];
    __shared__ float s_u[VNODES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid < a.T) {
        s_parent[tid] = tid ? a.parents[tid] : -1;
        s_token[tid] = a.tokens[tid];
        if (!GREEDY) s_u[tid] = a.uniforms[tid];
    }
    __syncthreads();
    for (int row = wave; row < a.T; row += VWALK / 64) {
        const float* pm = a.m + size_t(row) * a.chunks;
        float m = -__builtin_inff();
        for (int c = lane; c < a.chunks; c += 64) m = fmaxf(m, pm[c]);
        m = wave_max(m);
        if (GREEDY) {
            int at = a.V - 1;
            for (int c = lane; c < a.chunks; c += 64)
                if (pm[c] == m) at = min(at, reinterpret_cast<const int32_t*>(a.z)[size_t(row) * a.chunks + c]);
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) at = min(at, __shfl_xor(at, off, WAVE));
            if (lane == 0) s_best[row] = at;
            continue;
        }
        const double* pz = a.z + size_t(row) * a.chunks;
        double z = 0.0;
        for (int c = lane; c < a.chunks; c += 64) z += pz[c] * weight(pm[c], m, a.inv_t);
        z = wave_sum64(z);
        double ak = 1.0 / z, bk = 0.0;
        int level = 0;   // the last one that left something
        if (lane == 0) {
            s_m[row] = m;
            s_z[row] = z;
            s_a[row][0] = ak;
            s_b[row][0] = bk;
            s_level[row][0] = 0;
        }
        if (a.levels == 0) continue;
        const int kids = min(a.levels, int(__popcll(__ballot(lane < a.T && s_parent[min(lane, a.T - 1)] == row))));
        for (int l = 1; l <= kids; ++l) {
            const double* ps = a.s + (size_t(l - 1) * a.T + row) * a.chunks;
            double s = 0.0;
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
    __syncthreads();
    if (!GREEDY) {
        if (tid > 0 && tid < a.T) {
            const int p = s_parent[tid];
            const int64_t x = s_token[tid];
            const bool known = p >= 0 && p < tid && x >= 0 && x < a.V;
            s_e[tid] = known ? weight(logit<F32>(a.logits, size_t(p) * a.V + x), s_m[p], a.inv_t) : 0.0;
            s_q[tid] = known && a.draft ? double(a.draft[size_t(p) * a.V + x]) : 1.0;
        }
        __syncthreads();
    }
    if (tid == 0) {   // children come after their parents: one pass
        int cur = 0, n = 1, tried = 0, gone = 0;
        double left = GREEDY ? 0.0 : s_z[0];
        a.path[0] = 0;
        for (int c = 1; c < a.T; ++c) {
            if (s_parent[c] != cur) continue;
            bool take;
            if (GREEDY) {
                take = s_token[c] == s_best[cur];
            } else if (a.draft) {
                if (tried == a.levels) continue;
                const double r = fmax(s_a[cur][tried] * s_e[c] - s_b[cur][tried] * s_q[c], 0.0);
                take = double(s_u[c]) * s_q[c] < r;
                ++tried;
            } else {
                double e = s_e[c];
                for (int i = 0; i < gone; ++i)
                    if (s_token[s_gone[i]] == s_token[c]) e = 0.0;
                take = double(s_u[c]) * left < e;
                if (!take && e > 0.0 && left - e > 0.0) {
                    left -= e;
                    s_gone[gone++] = c;
                }
            }
            if (take) {
                cur = c;
                a.path[n++] = c;
                tried = gone = 0;
                left = GREEDY ? 0.0 : s_z[c];
            }
        }
        a.count[0] = n;
        for (int i = n; i < a.T; ++i) a.path[i] = -1;
        if (GREEDY) a.next[0] = s_best[cur];
        s_last = cur;
        s_lvl = tried;
        s_ngone = gone;
        s_lo = VWALK;
        s_hi = -1;
    }
    if (GREEDY) return;
    __syncthreads();
    const int cur = s_last, gone = s_ngone, lvl = s_level[cur][s_lvl];
    const float m = s_m[cur];
    double w = 0.0;
    if (tid < a.chunks) {
        if (lvl > 0) {
            w = a.s[(size_t(lvl - 1) * a.T + cur) * a.chunks + tid];
        } else {
            w = a.z[size_t(cur) * a.chunks + tid] * weight(a.m[size_t(cur) * a.chunks + tid], m, a.inv_t);
            for (int i = 0; i < gone; ++i)
                if (s_token[s_gone[i]] / VCHUNK == tid) w = fmax(w - s_e[s_gone[i]], 0.0);
        }
    }
    double upto = group_scan(w, s_wave);
    double total = 0.0;
    for (int i = 0; i < VWALK / 64; ++i) total = i ? total + s_wave[i] : s_wave[0];
    const double target = double(s_u[0]) * total;
    if (w > 0.0 && upto > target) atomicMin(&s_lo, tid);
    if (w > 0.0) atomicMax(&s_hi, tid);
    __syncthreads();
    const int chunk = s_lo < VWALK ? s_lo : max(s_hi, 0);   // (no sum above the target: the last chunk that has any)
    __syncthreads();
    if (tid == chunk) {
        s_z[0] = upto - w;
        s_lo = a.V;
        s_hi = -1;
    }
    __syncthreads();
    // the chunk again, four tokens a thread
    double part[4], sum = 0.0;
    const int v0 = chunk * VCHUNK + 4 * tid;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int v = v0 + i;
        double r = 0.0;
        if (v < a.V) {
            const double e = weight(logit<F32>(a.logits, size_t(cur) * a.V + v), m, a.inv_t);
            if (lvl > 0) {   // in the units of the level's sums, which stand before their normalisation
                r = fmax(s_a[cur][lvl - 1] * e - (s_b[cur][lvl - 1] + 1.0) * double(a.draft[size_t(cur) * a.V + v]), 0.0);
            } else {
                r = e;
                for (int j = 0; j < gone; ++j)
                    if (s_token[s_gone[j]] == v) r = 0.0;
            }
        }
        sum += r;
        part[i] = sum;
        if (r > 0.0) atomicMax(&s_hi, v);
    }
    const double before = s_z[0] + group_scan(sum, s_wave) - sum;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if ((i ? part[i] > part[i - 1] : part[i] > 0.0) && before + part[i] > target) atomicMin(&s_lo, v0 + i);
    __syncthreads();
    if (tid == 0) a.next[0] = s_lo < a.V ? s_lo : max(s_hi, 0);
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
    VerifyArgs a{tokens, parents, logits, greedy ? nullptr : draft, uniforms, path, count, next, T, V, chunks, levels, greedy ? 1.0 : 1.0 / temperature,
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
