// Products of MXFP4 operands (include/scmx_mx.h, scmx_mx_mm and scmx_mx_linear) on the scaled matrix instructions: v_mfma_scale_f32_32x32x64 and
// 16x16x128, both operands E2M1 with an E8M0 byte for 32 values, sums in float32.  The weights are the row operand, so that a lane's
// accumulators are groups of four consecutive columns n of one row m, two gates and their two ups among them.
//
// A lane's operand of either instruction is 16 bytes of codes, one block of 32 values, with the block's byte beside it.  Which blocks
// of K meet in an instruction is free, as long as both operands take the same.
#include <type_traits>

#include "mx.h"

namespace scmx {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct MxArgs {
    const uint8_t* x;
    const uint8_t* xs;
    const uint8_t* w;
    const uint8_t* ws;
    const uint16_t* res;
    uint16_t* out;
    int epi, M, N, K;
};

__device__ __forceinline__ i32x8 operand(u32x4 c) { return i32x8{int(c[0]), int(c[1]), int(c[2]), int(c[3]), 0, 0, 0, 0}; }
constexpr int FP4 = 4;   // of the instructions' format operands

__device__ __forceinline__ float silu_mul(float g, float u) {
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * g)) * u;
}

// Columns n .. n + 3 of row m (n a multiple of 4, both inside or past the ends).
__device__ __forceinline__ void store4(const MxArgs& a, int m, int n, const float* v) {
    if (m >= a.M || n >= a.N) return;
    if (a.epi == 3) {
        *reinterpret_cast<uint32_t*>(a.out + (size_t(m) * a.N + n) / 2) = f32_to_bf16x2(silu_mul(v[0], v[2]), silu_mul(v[1], v[3]));
        return;
    }
    const size_t at = size_t(m) * a.N + n;
    if (a.N % 4 == 0) {
        u32x2 r = {0, 0};
        if (a.epi == 2) r = *reinterpret_cast<const u32x2*>(a.res + at);
        *reinterpret_cast<u32x2*>(a.out + at) =
            a.epi == 2 ? u32x2{f32_to_bf16x2(v[0] + bf16_lo(r[0]), v[1] + bf16_hi(r[0])), f32_to_bf16x2(v[2] + bf16_lo(r[1]), v[3] + bf16_hi(r[1]))}
                       : u32x2{f32_to_bf16x2(v[0], v[1]), f32_to_bf16x2(v[2], v[3])};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < a.N) a.out[at + i] = f32_to_bf16(a.epi == 2 ? v[i] + bf16_to_f32(a.res[at + i]) : v[i]);
    }
}

// Few rows: a workgroup per 16 columns and 16 rows, its waves take the steps of 128 along K in turn, straight from memory.
constexpr int RWAVES = 4;
__global__ __launch_bounds__(64 * RWAVES) void mx_rows_kernel(const MxArgs a) {
    __shared__ f32x4 s_acc[RWAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ln = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16, nb = a.K / 32;
    const size_t wr = min(n0 + ln, a.N - 1), xr = min(m0 + ln, a.M - 1);
    const u32x4* wp = reinterpret_cast<const u32x4*>(a.w) + wr * nb;
    const u32x4* xp = reinterpret_cast<const u32x4*>(a.x) + xr * nb;
    const uint8_t *wsp = a.ws + wr * nb, *xsp = a.xs + xr * nb;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c0 = 4 * wave; c0 < nb; c0 += 4 * RWAVES) {
        const int c = c0 + g;
        u32x4 wc = {0, 0, 0, 0}, xc = {0, 0, 0, 0};
        int sw = 127, sx = 127;
        if (c < nb) {
            wc = wp[c];
            xc = xp[c];
            sw = wsp[c];
            sx = xsp[c];
        }
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(wc), operand(xc), acc, FP4, FP4, 0, sw, 0, sx);
    }
    s_acc[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < RWAVES; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += s_acc[w][lane][i];
    float v[4] = {acc[0], acc[1], acc[2], acc[3]};
    store4(a, m0 + ln, n0 + 4 * g, v);
}

// 16 bytes a lane past the registers: to lds + 16 * lane, zeros where `at` is behind the buffer's end.  (A function of its own: in a template
// the host's pass would drop the kernel.)
__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t from, uint8_t* lds, unsigned at) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)lds, 16, int(at), 0, 0, 0);
}

// Many rows: a workgroup of WM x WN waves per BM x BN tile.  A stage is 256 of K: BN + BM rows of 128 bytes of codes, loaded into LDS past the
// registers, 16 bytes a lane; chunk c of row r sits at chunk c ^ (r % 8), so that eight rows' chunks lie in different banks.  Rows and
// blocks behind the operands' ends are out of the buffers' bounds and come as zeros.  A lane of half h takes block 4 h + s in step s, so that
// the bytes of its four steps are one word, straight from memory.
template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 1) void mx_tile_kernel(const MxArgs a, int tiles_m, int tiles_n) {
    constexpr int NW = WM * WN, ROWS = BM + BN, STAGE = ROWS * 128, LOADS = ROWS / 8 / NW;
    constexpr int TI = BN / WN / 32, TJ = BM / WM / 32;   // a wave's blocks of 32 columns n, of 32 rows m
    static_assert(ROWS % (8 * NW) == 0 && BN % (8 * NW) == 0, "a wave loads whole pieces of one operand");
    __shared__ __attribute__((aligned(16))) uint8_t smem[2 * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, h = lane >> 5;
    const int wm = wave % WM, wn = wave / WM;
    const int m0 = int(blockIdx.x) % tiles_m * BM, n0 = int(blockIdx.x) / tiles_m * BN;
    const int nb = a.K / 32, steps = (nb + 7) / 8;
    const auto resource = [&](const uint8_t* p, int first, int rows, int most) {
        const int n = min(rows - first, most);
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p) + size_t(first) * nb * 16, 0, n * nb * 16, 0x00020000);
    };
    const auto wbuf = resource(a.w, n0, a.N, BN), xbuf = resource(a.x, m0, a.M, BM);
    const int r8 = lane / 8, chunk = (lane % 8) ^ r8;
    const auto load = [&](int step, int to) __attribute__((always_inline)) {
        const bool there = step * 8 + chunk < nb;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int piece = wave + NW * i, row = piece * 8;   // pieces of the weights first
            const bool of_w = row < BN;
            const unsigned at = there ? unsigned((of_w ? row : row - BN) + r8) * unsigned(nb * 16) + unsigned(step * 8 + chunk) * 16u : 0x7FFFFFF0u;
            uint8_t* lds = smem + to * STAGE + piece * 1024;
            if (of_w) load_lds16(wbuf, lds, at);
            else load_lds16(xbuf, lds, at);
        }
    };
    // The bytes of blocks 8 step + 4 h ..+ 3 of the lane's rows; bytes of blocks behind the end count as 127.
    const auto bytes = [&](const uint8_t* s, int row, int rows, int step) __attribute__((always_inline)) {
        const int64_t at = int64_t(min(row, rows - 1)) * nb + 8 * step + 4 * h, last = int64_t(rows) * nb - 4;
        const int64_t from = min(at, last);   // (the last word of the tensor holds its last bytes)
        typedef uint32_t u32u __attribute__((aligned(1)));
        uint32_t v = *reinterpret_cast<const u32u*>(s + from);
        if (8 * step + 8 > nb) {
            const int left = nb - 8 * step - 4 * h;
            v = at - from >= 4 ? 0 : v >> (8 * (at - from));
            if (left <= 0) v = 0x7F7F7F7Fu;
            else if (left < 4) v = (v & ((1u << (8 * left)) - 1)) | (0x7F7F7F7Fu << (8 * left));
        }
        return int(v);
    };
    f32x16 acc[TI][TJ];
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    load(0, 0);
    for (int step = 0; step < steps; ++step) {
        int sw[TI], sx[TJ];
#pragma unroll
        for (int i = 0; i < TI; ++i) sw[i] = bytes(a.ws, n0 + (wn * TI + i) * 32 + l32, a.N, step);
#pragma unroll
        for (int j = 0; j < TJ; ++j) sx[j] = bytes(a.xs, m0 + (wm * TJ + j) * 32 + l32, a.M, step);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();   // this stage has arrived, the other one is free
        if (step + 1 < steps) load(step + 1, (step + 1) & 1);
        const uint8_t* st = smem + (step & 1) * STAGE;
        const auto frag = [&](int row, int s) __attribute__((always_inline)) {
            return operand(*reinterpret_cast<const u32x4*>(st + row * 128 + (((4 * h + s) ^ (row & 7)) * 16)));
        };
        const auto part = [&](auto ss) __attribute__((always_inline)) {
            constexpr int S = decltype(ss)::value;
            i32x8 wf[TI], xf[TJ];
#pragma unroll
            for (int i = 0; i < TI; ++i) wf[i] = frag((wn * TI + i) * 32 + l32, S);
#pragma unroll
            for (int j = 0; j < TJ; ++j) xf[j] = frag(BN + (wm * TJ + j) * 32 + l32, S);
#pragma unroll
            for (int i = 0; i < TI; ++i)
#pragma unroll
                for (int j = 0; j < TJ; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[i], xf[j], acc[i][j], FP4, FP4, S, sw[i], S, sx[j]);
        };
        part(std::integral_constant<int, 0>{});
        part(std::integral_constant<int, 1>{});
        part(std::integral_constant<int, 2>{});
        part(std::integral_constant<int, 3>{});
    }
#pragma unroll
    for (int i = 0; i < TI; ++i)
#pragma unroll
        for (int j = 0; j < TJ; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float v[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                store4(a, m0 + (wm * TJ + j) * 32 + l32, n0 + (wn * TI + i) * 32 + 8 * q + 4 * h, v);
            }
}

template <int BM, int BN, int WM, int WN>
static void launch_tile(const MxArgs& a, hipStream_t st) {
    const int tm = (a.M + BM - 1) / BM, tn = (a.N + BN - 1) / BN;
    mx_tile_kernel<BM, BN, WM, WN><<<dim3(unsigned(tm) * unsigned(tn)), dim3(64 * WM * WN), 0, st>>>(a, tm, tn);
}

}  // namespace scmx

using namespace scmx;

static int check_mm(const char* who, const void* w, const void* ws, const void* res, const void* out, int epi, int M, int N, int K) {
    if (M < 0 || N < 1 || K < 32 || K % 32 || K > (1 << 23) || epi < 1 || epi > 3 || (epi == 3 && N % 4)) {
        set_error("%s: need epilogue 1..3, K a multiple of 32 up to 2^23 and for SwiGLU N a multiple of 4 (epi=%d M=%d N=%d K=%d)", who, epi, M, N, K);
        return SCMX_ERR_ARG;
    }
    if (M && (!w || !ws || !out || (epi == 2 && !res))) {
        set_error("%s: null pointer argument", who);
        return SCMX_ERR_ARG;
    }
    if ((uintptr_t(w) | uintptr_t(out) | uintptr_t(epi == 2 ? res : nullptr)) % 16) {
        set_error("%s: codes, res and out must be 16-byte aligned", who);
        return SCMX_ERR_ARG;
    }
    const int64_t tiles = ((int64_t(M) + 15) / 16) * ((int64_t(N) + 15) / 16);
    if (tiles > 0x7FFFFFFF) {
        set_error("%s: too many values out (M=%d N=%d)", who, M, N);
        return SCMX_ERR_ARG;
    }
    return SCMX_OK;
}

extern "C" int scmx_mx_mm(const uint8_t* xcodes, const uint8_t* xscales, const uint8_t* wcodes, const uint8_t* wscales, const uint16_t* res,
                          uint16_t* out, int epi, int M, int N, int K, void* stream) {
    if (int rc = check_mm("mx_mm", wcodes, wscales, res, out, epi, M, N, K)) return rc;
    if (M && (!xcodes || !xscales)) {
        set_error("mx_mm: null pointer argument");
        return SCMX_ERR_ARG;
    }
    if (uintptr_t(xcodes) % 16) {
        set_error("mx_mm: codes must be 16-byte aligned");
        return SCMX_ERR_ARG;
    }
    if (M == 0) return SCMX_OK;
    const MxArgs a{xcodes, xscales, wcodes, wscales, res, out, epi, M, N, K};
    const hipStream_t st = (hipStream_t)stream;
    const bool tiny = int64_t(K / 32) * (M < N ? M : N) < 4;   // (an operand has not four bytes of scales)
    if ((M <= 16 || tiny) && (M + 15) / 16 <= 65535) {
        mx_rows_kernel<<<dim3((N + 15) / 16, (M + 15) / 16), dim3(64 * RWAVES), 0, st>>>(a);
    } else if (int64_t(M) * N >= int64_t(256) * 256 * 200) {
        launch_tile<256, 256, 2, 2>(a, st);
    } else if (int64_t(M) * N >= int64_t(128) * 128 * 128) {
        launch_tile<128, 128, 2, 2>(a, st);
    } else {
        launch_tile<64, 64, 2, 2>(a, st);
    }
    return check_launch("mx_mm");
}

extern "C" size_t scmx_mx_linear_workspace(int M, int N, int K) {
    if (M < 1 || N < 1 || K < 32 || K % 32) return 0;
    return size_t(M) * (K / 2) + size_t(M) * (K / 32);
}

extern "C" int scmx_mx_linear(const uint16_t* x, int64_t ldx, const uint16_t* nw, float eps, const uint8_t* wcodes, const uint8_t* wscales,
                              const uint16_t* res, uint16_t* out, int epi, int M, int N, int K, void* workspace, size_t workspace_bytes,
                              void* stream) {
    if (int rc = check_mm("mx_linear", wcodes, wscales, res, out, epi, M, N, K)) return rc;
    const size_t need = scmx_mx_linear_workspace(M, N, K);
    if (workspace_bytes < need || (need && !workspace) || uintptr_t(workspace) % 16) {
        set_error("mx_linear: needs a 16-byte aligned workspace of %zu bytes", need);
        return SCMX_ERR_WORKSPACE;
    }
    uint8_t *codes = static_cast<uint8_t*>(workspace), *scales = codes + size_t(M) * (K / 2);
    if (int rc = scmx_mx_quantize(x, SCMX_MX_BF16, ldx, nw, eps, codes, scales, M, K, stream)) return rc;
    return scmx_mx_mm(codes, scales, wcodes, wscales, res, out, epi, M, N, K, stream);
}
