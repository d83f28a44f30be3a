// Products of MXFP4 operands (include/scmx_mx.h, scmx_mx_mm and scmx_mx_linear) on the scaled matrix instructions:
// v_mfma_scale_f32_16x16x128, both operands E2M1 with an E8M0 byte for 32 values, sums in float32.  The weights are the row operand, so
// that a lane's accumulators are groups of four consecutive columns n of one row m, two gates and their two ups among them.
//
// A lane's operand is 16 bytes of codes, one block of 32 values, with the block's byte beside it.  Which blocks
// of K meet in an instruction is free, as long as both operands take the same.
#include <type_traits>

#include "mx.h"

namespace scmx {

typedef int i32x8 __attribute__((ext_vector_type(8)));

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
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));   // (the hardware takes vectors at any address)
typedef uint32_t u32x4b __attribute__((ext_vector_type(4), aligned(1)));

__device__ __forceinline__ float silu_mul(float g, float u) {
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * g)) * u;
}

// Columns n .. n + 3 of row m, those that are inside (n is a multiple of 4); one by one where rows are no multiple of 4.
template <int EPI>
__device__ __forceinline__ void store4(const MxArgs& a, int m, int n, f32x4 v) {
    if (m >= a.M) return;
    if constexpr (EPI == 3) {
        if (n < a.N)
            *reinterpret_cast<uint32_t*>(a.out + (size_t(m) * a.N + n) / 2) = f32_to_bf16x2(silu_mul(v[0], v[2]), silu_mul(v[1], v[3]));
    } else {
        const size_t at = size_t(m) * a.N + n;
        if (a.N % 4 == 0) {
            if (n >= a.N) return;
            if constexpr (EPI == 2) {
                const u32x2 r = *reinterpret_cast<const u32x2*>(a.res + at);
                v = f32x4{v[0] + bf16_lo(r[0]), v[1] + bf16_hi(r[0]), v[2] + bf16_lo(r[1]), v[3] + bf16_hi(r[1])};
            }
            *reinterpret_cast<u32x2*>(a.out + at) = u32x2{f32_to_bf16x2(v[0], v[1]), f32_to_bf16x2(v[2], v[3])};
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < a.N) a.out[at + i] = f32_to_bf16(EPI == 2 ? v[i] + bf16_to_f32(a.res[at + i]) : v[i]);
    }
}

// Columns n .. n + 7 (SwiGLU: n + 15) of row m, all inside, in one store of eight values; a row starts at any even address (the hardware
// takes vectors at them).
template <int EPI>
__device__ __forceinline__ void store(const MxArgs& a, int m, int n, const float* v) {
    const size_t at = EPI == 3 ? (size_t(m) * a.N + n) / 2 : size_t(m) * a.N + n;
    u32x4 r = {0, 0, 0, 0}, w;
    if constexpr (EPI == 2) r = *reinterpret_cast<const u32x4u*>(a.res + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (EPI == 1) w[i] = f32_to_bf16x2(v[2 * i], v[2 * i + 1]);
        else if constexpr (EPI == 2) w[i] = f32_to_bf16x2(v[2 * i] + bf16_lo(r[i]), v[2 * i + 1] + bf16_hi(r[i]));
        else w[i] = f32_to_bf16x2(silu_mul(v[4 * i], v[4 * i + 2]), silu_mul(v[4 * i + 1], v[4 * i + 3]));
    }
    *reinterpret_cast<u32x4u*>(a.out + at) = w;
}

// Few rows: a workgroup per 16 columns (8 where the workgroups would be too few: half of a fragment's columns are none then) and 16
// rows.  BLOCKS of K at a time, the rows' codes come to LDS, as they are or made of bf16 rows (a thread takes a block of 32, 64 bytes,
// and needs no other's values), and the waves take steps of 128 side by side, the weights straight from memory, requested before the
// rows.  The waves meet in LDS.  Bound by reading the weights where there are many (16384 x 8192 17.9-19.1 us, 3.7-4.0 TB/s), by the
// launch and a trip to memory where there are few.
constexpr int FEW_WAVES = 8;

struct FewArgs : MxArgs {
    const uint16_t* rows;   // NULL: codes
    int64_t ldx;
};

// The operand and byte of a block of 32 bf16 values.
__device__ __forceinline__ u32x4 block_codes(const u32x4 (&v)[4], uint32_t& byte) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 top = {0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, v[i / 4][i % 4] & 0x7FFF7FFFu));
    byte = mx_byte(uint32_t(max(top[0], top[1])) << 16);
    u32x4 c;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = mx_codes_bf16(v[i], byte);
    return c;
}

template <int COLS, int BLOCKS>
__global__ __launch_bounds__(64 * FEW_WAVES) void mx_few_kernel(const FewArgs a) {
    constexpr int WAVES = FEW_WAVES, U = BLOCKS / 4 / WAVES;   // steps of a wave, whose loads are on their way together
    __shared__ f32x4 s_acc[WAVES][64];
    __shared__ u32x4 s_x[16][BLOCKS + 1];   // (rows' blocks in different banks)
    __shared__ uint8_t s_xs[16][BLOCKS + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), ln = lane & 15, g = lane >> 4;
    const unsigned down = (blockIdx.z * gridDim.y + blockIdx.y) * 16;
    if (down >= unsigned(a.M)) return;
    const int n0 = blockIdx.x * COLS, m0 = int(down), nb = a.K / 32, high = min(a.M - m0, 16), row = min(ln, high - 1);
    const size_t wr = min(n0 + ln, a.N - 1);
    const u32x4* wp = reinterpret_cast<const u32x4*>(a.w) + wr * nb;
    const uint8_t* wsp = a.ws + wr * nb;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int b0 = 0; b0 < nb; b0 += BLOCKS) {
        const int blocks = min(nb - b0, BLOCKS), per = ((blocks + 3) / 4 + WAVES - 1) / WAVES, first = wave * per;
        u32x4 wc[U];
        uint32_t sw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = 4 * (first + u) + g;
            const bool there = u < per && c < blocks && ln < COLS;
            wc[u] = there ? wp[b0 + c] : u32x4{0, 0, 0, 0};
            sw[u] = there ? wsp[b0 + c] : 0;
        }
        if (b0) __syncthreads();   // (all have read the blocks before)
        for (int i = tid; i < high * blocks; i += 64 * WAVES) {
            const int r = unsigned(i) / unsigned(blocks), c = i - r * blocks;
            if (a.rows) {
                const u32x4u* p = reinterpret_cast<const u32x4u*>(a.rows + (m0 + r) * a.ldx + 32 * (b0 + c));
                const u32x4 v[4] = {p[0], p[1], p[2], p[3]};
                uint32_t byte;
                s_x[r][c] = block_codes(v, byte);
                s_xs[r][c] = uint8_t(byte);
            } else {
                const size_t at = size_t(m0 + r) * nb + b0 + c;
                s_x[r][c] = reinterpret_cast<const u32x4*>(a.x)[at];
                s_xs[r][c] = a.xs[at];
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= per) break;
            const int c = min(4 * (first + u) + g, blocks - 1);   // (behind the end: a block that meets zeros, its byte with them)
            const uint32_t sx = 4 * (first + u) + g < blocks ? s_xs[row][c] : 0;
            acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(wc[u]), operand(s_x[row][c]), acc, FP4, FP4, 0, int(sw[u]), 0,
                                                                   int(sx));
        }
    }
    s_acc[wave][lane] = acc;
    __syncthreads();
    if (wave || 4 * g >= COLS) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += s_acc[w][lane][i];
    if (a.epi == 1) store4<1>(a, m0 + ln, n0 + 4 * g, acc);
    else if (a.epi == 2) store4<2>(a, m0 + ln, n0 + 4 * g, acc);
    else store4<3>(a, m0 + ln, n0 + 4 * g, acc);
}

// 16 bytes a lane past the registers: to LDS byte `lds` + 16 * lane, zeros where `at` is behind the buffer's end.  Written out because the
// compiler, which cannot tell one stage's place from another's, would wait for all such loads before each read of LDS; who reads what
// they bring waits for them itself.  (m0 is the place; a state between its setting and its use.)
typedef uint32_t Buffer __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void load_lds16(Buffer from, unsigned lds, unsigned at) {
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "{m0}"(lds), "v"(at), "s"(from) : "memory");
}
__device__ __forceinline__ Buffer buffer_of(const uint8_t* p, unsigned bytes) {
    const uint64_t at = reinterpret_cast<uint64_t>(p);
    return Buffer{uint32_t(__builtin_amdgcn_readfirstlane(int(at))), uint32_t(__builtin_amdgcn_readfirstlane(int(at >> 32))) & 0xFFFFu,
                  uint32_t(__builtin_amdgcn_readfirstlane(int(bytes))), 0x00020000u};
}
__device__ __forceinline__ unsigned lds_offset(const uint8_t* p) {
    return unsigned(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t*)p));
}

// acc += w x in place, step S's bytes of sw and sx.  Written out because the compiler otherwise moves accumulators between registers all
// through a loop that leaves it none.  What it would add by itself: two states between a vector instruction's write of an operand and
// this (`settle`), and eighteen between this and a read of acc by anything else (`done`); loads of operands it waits for by itself.
template <int S>
__device__ __forceinline__ void multiply(f32x4& acc, u32x4 w, u32x4 x, int sw, int sx) {
    if constexpr (S == 0)
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                     : "+a"(acc) : "v"(w), "v"(x), "v"(sw), "v"(sx));
    else
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                     : "+a"(acc) : "v"(w), "v"(x), "v"(sw), "v"(sx));
}
__device__ __forceinline__ void settle() { asm volatile("s_nop 1"); }
__device__ __forceinline__ void done() { asm volatile("s_nop 15\n\ts_nop 3"); }

// Many rows: workgroups of 2 x 2 waves take BM x BN tiles in turn.  A stage is 256 of K: BN + BM rows of 128 bytes of codes, loaded into
// LDS past the registers, 16 bytes a lane; chunk c (a block of 32) of row r sits at chunk (c % 2 * 4 + c / 2) ^ (r / 2 % 8), so that a
// fragment's lanes find theirs in different banks.  Rows and blocks behind the operands' ends are out of the buffers' bounds and come as
// zeros.  In step s of a stage's two, lane group g takes block 2 g + s, so that its bytes lie side by side.  The bytes of four stages
// come together, 32 a row.
//
// Two stages: half way through one, its second step's fragments are in registers and the next stage has arrived (one barrier says both);
// its place is loaded with the stage after the next, of the next tile too, while the second step multiplies, and the next stage's first
// fragments are read.  So a tile's results are written while the next one's operands are on their way.
//
// Row p of the weights' part of LDS is a column of the tile such that Q fragments' accumulators (four for SwiGLU, else two) are 4 Q
// consecutive columns of a lane, and the four lane groups' stores 64 bytes of a row.
template <int BM, int BN, int EPI, bool EVEN>
__global__ __launch_bounds__(256, 1) void mx_tile_kernel(const MxArgs a, int tiles_m, int tiles_n) {
    constexpr int NW = 4, ROWS = BM + BN, STAGE = ROWS * 128, LOADS = ROWS / 8 / NW, WLOADS = BN / 8 / NW;
    constexpr int TI = BN / 2 / 16, TJ = BM / 2 / 16;   // a wave's blocks of 16 columns n, of 16 rows m
    constexpr int SROWS = ROWS * 32, READS = TI + TJ, Q = EPI == 3 ? 4 : 2;
    constexpr int STORES = TI / Q * TJ;                 // a wave's stores of a whole tile
    static_assert((BM == 32 || BM % 64 == 0) && BM <= 256 && BN % 128 == 0 && BN <= 256,
                  "a wave loads whole pieces of one operand and holds 64 columns' fragments");
    static_assert(READS == LOADS && STORES < 64, "as many fragments a step as pieces a stage; a counter of six bits");
    __shared__ __attribute__((aligned(16))) uint8_t smem[2 * STAGE], s_scale[2 * SROWS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), ln = lane & 15, g = lane >> 4;
    const int wm = wave % 2, wn = wave / 2;
    // In a round of all workgroups a run of tiles to each XCD (workgroups are dealt to them in turn), in strips of eight tile rows
    const int all = tiles_m * tiles_n, grid = int(gridDim.x), b = int(blockIdx.x);
    const int mine = grid % 8 == 0 ? b % 8 * (grid / 8) + b / 8 : b;
    const auto tile_m = [&](int o) {
        const int strip = o / (8 * tiles_n), high = min(8, tiles_m - 8 * strip);
        return (8 * strip + (o - strip * 8 * tiles_n) % high) * BM;
    };
    const auto tile_n = [&](int o) {
        const int strip = o / (8 * tiles_n), high = min(8, tiles_m - 8 * strip);
        return (o - strip * 8 * tiles_n) / high * BN;
    };
    const int nb = a.K / 32, stages = (nb + 7) / 8;
    // row p of LDS: which row of its operand's part of the tile
    const auto source = [](int p) { return p < BN ? p / (16 * Q) * (16 * Q) + p % 16 / 4 * (4 * Q) + p / 16 % Q * 4 + p % 4 : p - BN; };
    // offsets of blocks from nb on get the top bit, which no buffer reaches (K <= 2^23: a tile's rows take up to 2^30 bytes)
    const auto behind = [&](int c) { return unsigned(nb - 1 - c) & 0x80000000u; };
    const unsigned codes_at = lds_offset(smem), scales_at = lds_offset(s_scale), row_bytes = unsigned(nb) * 16u;
    // pieces of eight rows, wave's wave + 4 i; the lane's 16 bytes in a row of each
    const int r8 = lane / 8, slot = (lane % 8) ^ (4 * (wave & 1) + r8 / 2), chunk = slot % 4 * 2 + slot / 4;
    const unsigned wlane = unsigned(source(8 * wave + r8)) * row_bytes + 16u * chunk;
    const unsigned xlane = unsigned(8 * wave + r8) * row_bytes + 16u * chunk;
    // of scales waves 0 and 1 bring the weights', 2 and 3 the rows', 32 rows a piece
    const bool of_w = wave < 2;
    const int odd = of_w || BM > 32 ? wave & 1 : 0;
    const int p0 = 32 * odd + lane / 2, half = 16 * (lane % 2 ^ (p0 / 8 & 1)), row0 = of_w ? source(p0) : p0;
    const unsigned scales_to = (of_w ? 0 : BN * 32) + odd * 1024, slane = unsigned(row0) * unsigned(nb) + half;
    // what is loaded next: stage l of tile lo; the bytes loaded last went to place lq % 2
    int lo = mine, l = 0, lq = -1;
    Buffer wbuf, xbuf, sbuf;
    const auto buffers = [&]() __attribute__((always_inline)) {
        const int m0 = tile_m(lo), n0 = tile_n(lo), first = of_w ? n0 : m0, rows = of_w ? min(a.N - n0, BN) : min(a.M - m0, BM);
        wbuf = buffer_of(a.w + size_t(n0) * row_bytes, unsigned(min(a.N - n0, BN)) * row_bytes);
        xbuf = buffer_of(a.x + size_t(m0) * row_bytes, unsigned(min(a.M - m0, BM)) * row_bytes);
        sbuf = buffer_of((of_w ? a.ws : a.xs) + size_t(first) * nb, unsigned(rows) * unsigned(nb));
    };
    const auto load = [&](int place, int i) __attribute__((always_inline)) {   // piece i of LOADS
        const unsigned to = codes_at + place * STAGE + wave * 1024 + i * 4096;
        const unsigned k = unsigned(l) * 128u | behind(l * 8 + chunk);
        // (row 32 i + .. of LDS is row 32 i + .. of the weights for Q = 2, row 64 (i / 2) + 8 (i % 2) + .. for Q = 4)
        if (i < WLOADS) load_lds16(wbuf, to, wlane + k + unsigned(Q == 2 ? 32 * i : i / 2 * 64 + i % 2 * 8) * row_bytes);
        else load_lds16(xbuf, to, xlane + k + unsigned(i - WLOADS) * 32u * row_bytes);
    };
    // The bytes of stages l .. l + 3; rows of bytes at any alignment come through the registers, and to LDS by put_scales.
    constexpr int PARTS = (BN > BM ? BN : BM) / 64;
    u32x4 held[EVEN ? 1 : PARTS];
    int over[EVEN ? 1 : PARTS];   // bytes that they are behind what is held
    bool holds = false;
    const auto parts = [&](auto&& go) __attribute__((always_inline)) {
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
            if (part < (of_w ? BN / 64 : BM == 32 ? 1 : BM / 64)) go(part, (lq & 1) * SROWS + scales_to + part * 2048);
    };
    const auto load_scales = [&]() __attribute__((always_inline)) {
        const int c = 4 * l * 2 + half;
        ++lq;
        parts([&](int part, unsigned to) __attribute__((always_inline)) {
            if constexpr (EVEN) {
                load_lds16(sbuf, scales_at + to, (slane + 8u * l + part * 64u * unsigned(nb)) | behind(c));
            } else {
                const int rows = of_w ? a.N : a.M, row = min((of_w ? tile_n(lo) : tile_m(lo)) + 64 * part + row0, rows - 1);
                const int64_t first = int64_t(row) * nb + c;
                const int64_t at = min(first, int64_t(rows) * nb - 16);   // (the last 16 hold the last bytes)
                held[part] = *reinterpret_cast<const u32x4b*>((of_w ? a.ws : a.xs) + at);
                over[part] = int(min(first - at, int64_t(16)));
            }
        });
        holds = !EVEN;
    };
    const auto put_scales = [&]() __attribute__((always_inline)) {
        if (EVEN || !holds) return;
        holds = false;
        parts([&](int part, unsigned to) __attribute__((always_inline)) {
            u32x4 v = held[part];
            if (__any(over[part])) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    uint32_t two[2] = {0, 0};   // the words that hold word u's bytes
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (i == u + over[part] / 4) two[0] = held[part][i];
                        if (i == u + over[part] / 4 + 1) two[1] = held[part][i];
                    }
                    v[u] = uint32_t((uint64_t(two[1]) << 32 | two[0]) >> (8 * (over[part] % 4)));
                }
            }
            *reinterpret_cast<u32x4*>(s_scale + to + 16 * lane) = v;
        });
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    const auto loaded = [&]() __attribute__((always_inline)) {   // on to the next stage
        if (++l < stages) return;
        l = 0;
        lo += grid;
        if (lo >= all) lo = all - 1;   // (behind the last tile: some tile, for nobody)
        buffers();
    };
    f32x4 acc[TI][TJ];
    u32x4 wf[2][TI], xf[2][TJ];   // the fragments of a stage's two steps
    int sw[TI], sx[TJ], sw_next[TI], sx_next[TJ];   // the bytes of both, and of the next stage's
    int place = 0, quad = 0;   // where in LDS the present stage and its bytes are
    const auto read = [&](int from, int r, int s) __attribute__((always_inline)) {   // fragment r of READS of step s
        const uint8_t* at = smem + from * STAGE + (((4 * s + g) ^ (ln / 2)) * 16) + ln * 128;
        if (r == 0) wf[s][0] = *reinterpret_cast<const u32x4*>(at + wn * TI * 2048);
        else if (r <= TJ) xf[s][r - 1] = *reinterpret_cast<const u32x4*>(at + BN * 128 + (wm * TJ + r - 1) * 2048);
        else wf[s][r - TJ] = *reinterpret_cast<const u32x4*>(at + (wn * TI + r - TJ) * 2048);
    };
    const auto read_scale = [&](int stage, int from, int r) __attribute__((always_inline)) {
        const uint8_t* at = s_scale + from * SROWS + ((stage % 4 * 8 + 2 * g) ^ (ln / 8 * 16)) + ln * 32;
        if (r < TI) sw_next[r] = *reinterpret_cast<const uint16_t*>(at + (wn * TI + r) * 512);
        else sx_next[r - TI] = *reinterpret_cast<const uint16_t*>(at + BN * 32 + (wm * TJ + r - TI) * 512);
    };
    // The instructions of a step, and before them one after the other the `items` of item(0 ..), done when three quarters of the step are:
    // a wave issues in order, and loads in a row would hold up the multiplications.
    const auto step = [&](auto ss, auto items, auto&& item) __attribute__((always_inline)) {
        constexpr int S = decltype(ss)::value, L = decltype(items)::value, N = TI * TJ, SPREAD = N * 3 / 4;
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
            for (int i = n * L / SPREAD; i < (n + 1) * L / SPREAD && i < L; ++i) item(i);
            __builtin_amdgcn_sched_barrier(0);
            multiply<S>(acc[n / TJ][n % TJ], wf[S][n / TJ], xf[S][n % TJ], sw[n / TJ], sx[n % TJ]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    const auto barrier = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    buffers();
    load_scales();
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load(0, i);
    loaded();
    put_scales();
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    barrier();
    if (l % 4 == 0) load_scales();
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load(1, i);
    loaded();
#pragma unroll
    for (int r = 0; r < READS; ++r) read(0, r, 0);
#pragma unroll
    for (int r = 0; r < READS; ++r) read_scale(0, 0, r);
    bool stores = false;   // of a whole tile are on their way
    for (int o = mine; o < all; o += grid) {
        const int m0 = tile_m(o), n0 = tile_n(o);
#pragma unroll
        for (int i = 0; i < TI; ++i)
#pragma unroll
            for (int j = 0; j < TJ; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int t = 0; t < stages; ++t) {
            // bytes of blocks behind the end are another row's: their codes are zeros, a NaN they must not be
            const int left = nb - 8 * t - 2 * g, keep = left >= 2 ? 0xFFFF : left == 1 ? 0xFF : 0;
#pragma unroll
            for (int i = 0; i < TI; ++i) sw[i] = sw_next[i] & keep;
#pragma unroll
            for (int j = 0; j < TJ; ++j) sx[j] = sx_next[j] & keep;
            settle();
            __builtin_amdgcn_sched_barrier(0);
            step(std::integral_constant<int, 0>{}, std::integral_constant<int, READS>{},
                 [&](int i) __attribute__((always_inline)) { read(place, i, 1); });
            // every wave has read this stage whole, and the next one is there: its loads are older than the last tile's stores
            if (t == 0 && stores) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(STORES) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            put_scales();
            barrier();
            // the stage after it into this one's place; the next one's first fragments
            const int next = t + 1 < stages ? t + 1 : 0;
            if (next % 4 == 0) quad ^= 1;
            constexpr std::integral_constant<int, LOADS + 1 + 2 * READS> items;
            step(std::integral_constant<int, 1>{}, items, [&](int i) __attribute__((always_inline)) {
                if (i < 2 * LOADS) {
                    if (i % 2 == 0) load(place, i / 2);
                    else read(place ^ 1, i / 2, 0);
                } else if (i == 2 * LOADS) {
                    if constexpr (EVEN)
                        if (l % 4 == 0) load_scales();
                } else {
                    read_scale(next, quad, i - 2 * LOADS - 1);
                }
            });
            if constexpr (!EVEN)
                if (l % 4 == 0) load_scales();
            loaded();
            place ^= 1;
        }
        done();
        __builtin_amdgcn_sched_barrier(0);
        if (BM + BN == 512 || n0 + BN <= a.N || a.N % 16 == 0) {   // (the largest tile takes no other N: no registers for it)
            stores = m0 + BM <= a.M && n0 + BN <= a.N;   // (as many as counted)
#pragma unroll
            for (int j = 0; j < TJ; ++j) {
                int m = m0 + (wm * TJ + j) * 16 + ln;
                asm volatile("" : "+v"(m));   // (registers for one row's results at a time)
#pragma unroll
                for (int i = 0; i < TI; i += Q) {
                    float v[4 * Q];
#pragma unroll
                    for (int r = 0; r < 4 * Q; ++r) v[r] = acc[i + r / 4][j][r % 4];
                    const int n = n0 + (wn * TI + i) * 16 + 4 * Q * g;
                    if (m < a.M && n < a.N) store<EPI>(a, m, n, v);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {   // the last columns of a number that is no multiple of 16: a fragment's four at a time
            stores = false;
#pragma unroll
            for (int j = 0; j < TJ; ++j) {
#pragma unroll
                for (int i = 0; i < TI; ++i)
                    store4<EPI>(a, m0 + (wm * TJ + j) * 16 + ln, n0 + source((wn * TI + i) * 16 + 4 * g), acc[i][j]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // (what was loaded for nobody: not into the next workgroup's LDS)
}

template <typename F>
static void by_epilogue(int epi, F&& go) {
    if (epi == 1) go(std::integral_constant<int, 1>{});
    else if (epi == 2) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 3>{});
}
template <int COLS, int BLOCKS>
static void few(const FewArgs& a, hipStream_t st) {
    const unsigned down = (unsigned(a.M) + 15) / 16, z = (down + 65534) / 65535;
    mx_few_kernel<COLS, BLOCKS><<<dim3((unsigned(a.N) + COLS - 1) / COLS, (down + z - 1) / z, z), dim3(64 * FEW_WAVES), 0, st>>>(a);
}
// Eight columns where that leaves no CU two workgroups.  us with 16 columns and 128 blocks / 16 and 256 / 8 and 256: one row of 12288 x
// 2048 4.9 / 6.9 / 7.7, of 16384 x 8192 20.1 / 17.9 / 20.0, of 4096 x 4096 4.1 / 4.2 / 4.5, of 2944 x 6752 4.3 / 4.2 / 4.9, of 2048 x
// 8192 6.1 / 5.9 / 4.5, 16 rows of 12288 x 2048 5.6 / 7.7 / 9.0, of 2048 x 8192 7.8 / 7.8 / 6.7.  16 waves: between these; 64 blocks: no
// better.
static void launch_few(const FewArgs& a, hipStream_t st) {
    if ((int64_t(a.N) + 15) / 16 * ((int64_t(a.M) + 15) / 16) <= device_cus() / 2) few<8, 256>(a, st);
    else if (a.K > 4096) few<16, 256>(a, st);
    else few<16, 128>(a, st);
}
// Whether every row's bytes are whole words.
static bool words(const MxArgs& a) {
    return a.K % 128 == 0 && (reinterpret_cast<uintptr_t>(a.xs) | reinterpret_cast<uintptr_t>(a.ws)) % 4 == 0;
}

template <int BM, int BN>
static void launch_tile(const MxArgs& a, hipStream_t st) {
    const int tm = int((unsigned(a.M) + BM - 1) / BM), tn = int((unsigned(a.N) + BN - 1) / BN);
    const unsigned tiles = unsigned(tm) * unsigned(tn), most = unsigned(device_cus()) * (BM + BN <= 256 ? 2 : 1);   // (as LDS holds)
    const dim3 grid(tiles < most ? tiles : most);
    by_epilogue(a.epi, [&](auto epi) {
        constexpr int EPI = decltype(epi)::value;
        if (BM + BN == 512 || words(a)) mx_tile_kernel<BM, BN, EPI, true><<<grid, dim3(256), 0, st>>>(a, tm, tn);
        else if constexpr (BM + BN < 512) mx_tile_kernel<BM, BN, EPI, false><<<grid, dim3(256), 0, st>>>(a, tm, tn);
    });
}

}  // namespace scmx

using namespace scmx;

constexpr int FEW = 16;   // rows up to which they are few

static int check_mm(const char* who, const void* w, const void* ws, const void* res, const void* out, int epi, int M, int N, int K) {
    if (M < 0 || N < 1 || K < 32 || K % 32 || K > (1 << 23) || epi < 1 || epi > 3 || (epi == 3 && N % 4)) {
        set_error("%s: need epilogue 1..3, K a multiple of 32 up to 2^23 and for SwiGLU N a multiple of 4 (epi=%d M=%d N=%d K=%d)", who,
                  epi, M, N, K);
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

// The tile that takes the least time, in us: alone on a CU a stage of 256 of K and a tile's beginning and end take so long, and so long
// for each tile when every CU has some (a CU that holds several takes them in turn or side by side alike); measured from 17 to 8192 rows,
// 512 to 16384 columns, K from 256 to 8192, where the choice is half a per cent off the best on average.  us for 32x128 / 64x128 /
// 128x128 / 256x256: 100 rows of 12288 x 2048 7.8 / 7.2 / 8.5 / 16.9, 333 of 5120 x 2944 11.2 / 9.6 / 11.0 / 24.5, 700 of 5120 x 2944
// 20.6 / 14.3 / 12.8 / 28.4, 6000 of 12288 x 2048 180 / 124 / 92 / 89, of 2048 x 8192 114 / 70 / 74 / 56, 4000 of 16384 x 512 58 / 44 /
// 35 / 46.
// Some rows go to the kernel of few, 16 at a time, where its workgroups are few too (us with tiles / with it: 17 rows of 2048 x 2048 5.9 /
// 3.5, of 4096 x 4096 8.6 / 6.7, of 12288 x 2048 6.1 / 9.0, 64 rows of 2048 x 2048 6.1 / 4.5, of 2048 x 8192 14.2 / 11.9, of 4096 x 4096
// 8.8 / 12.2, 333 of 512 x 2048 6.0 / 5.7).
constexpr int NO_TILE = 4;
static int tile_of(int M, int N, int K, bool words) {
    constexpr int BM[4] = {32, 64, 128, 256}, BN[4] = {128, 128, 128, 256};
    constexpr double ALONE[4] = {0.34, 0.35, 0.49, 1.1}, ALONE_ENDS[4] = {1.1, 1.4, 1.8, 5.2};
    constexpr double FULL[4] = {0.25, 0.34, 0.5, 1.4}, FULL_ENDS[4] = {0.45, 0.82, 1.2, 7.5};
    const int cus = device_cus(), most = N % 16 || !words ? 3 : 4;   // (the largest takes whole groups of columns and words of bytes)
    const double stages = (K + 255) / 256, groups = double((int64_t(M) + 15) / 16) * double((int64_t(N) + 15) / 16) / cus;
    int best = NO_TILE;
    double least = (groups < 1 ? 1 : groups) * (0.135 * stages + 0.33);
    for (int i = 0; i < most; ++i) {
        const int64_t tiles = (int64_t(M) + BM[i] - 1) / BM[i] * ((int64_t(N) + BN[i] - 1) / BN[i]);
        const double load = tiles < cus ? double(tiles) / cus : double((tiles + cus - 1) / cus);
        const double alone = (ALONE[i] + (words ? 0 : 0.13)) * stages + ALONE_ENDS[i];
        const double full = ((FULL[i] + (words ? 0 : 0.08)) * stages + FULL_ENDS[i]) * load;
        const double us = alone > full ? alone : full;
        if (us < least) {
            least = us;
            best = i;
        }
    }
    return best;
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
    const bool tiny = int64_t(K / 32) * (M < N ? M : N) < 16;   // (an operand has not sixteen bytes of scales)
    const int tile = M <= FEW || tiny ? NO_TILE : tile_of(M, N, K, words(a)), most = 0x7FFFFE00;
    if (tile == NO_TILE ? N > 1 << 26 : M > most || N > most) {   // (a tile's rows and columns behind the last are numbers too)
        set_error("mx_mm: too many rows or columns (M=%d N=%d)", M, N);
        return SCMX_ERR_ARG;
    }
    switch (tile) {
        case 0: launch_tile<32, 128>(a, st); break;
        case 1: launch_tile<64, 128>(a, st); break;
        case 2: launch_tile<128, 128>(a, st); break;
        case 3: launch_tile<256, 256>(a, st); break;
        default: {
            FewArgs f{};
            static_cast<MxArgs&>(f) = a;
            launch_few(f, st);
        }
    }
    return check_launch("mx_mm");
}

// Whether a linear layer's rows are quantised in the product's own kernel, that of few: every workgroup of its columns does it for
// itself, which costs a launch less and reads the rows N / 16 times.  us in one / in two: a row of 4096 x 4096 (2^24 products) 4.4 / 6.6,
// 16 rows of 4096 x 4096 (2^28) 6.4 / 8.1, of 12288 x 2048 (2^28.6) 8.1 / 9.3, 8 rows of 16384 x 4096 (2^29) 14.0 / 14.1, 16 (2^30) 18.1
// / 15.9, 64 rows of 2048 x 2048 (2^28) 6.3 / 7.4, 32 of 2048 x 8192 (2^29) 10.5 / 11.7, of 4096 x 4096 10.2 / 9.9, 64 of 2048 x 8192
// (2^30) 18.3 / 15.5.
static bool in_one(int M, int N, int K) {   // (bytes off a word only turn more to that kernel)
    return int64_t(M) * N <= (int64_t(1) << 29) / K && (M <= FEW || tile_of(M, N, K, K % 128 == 0) == NO_TILE);
}

extern "C" size_t scmx_mx_linear_workspace(int M, int N, int K, int norm) {
    if (M < 1 || N < 1 || K < 32 || K % 32 || (!norm && in_one(M, N, K))) return 0;
    return size_t(M) * (K / 2) + size_t(M) * (K / 32);
}

extern "C" int scmx_mx_linear(const uint16_t* x, int64_t ldx, const uint16_t* nw, float eps, const uint8_t* wcodes, const uint8_t* wscales,
                              const uint16_t* res, uint16_t* out, int epi, int M, int N, int K, void* workspace, size_t workspace_bytes,
                              void* stream) {
    if (int rc = check_mm("mx_linear", wcodes, wscales, res, out, epi, M, N, K)) return rc;
    const size_t need = scmx_mx_linear_workspace(M, N, K, nw != nullptr);
    if (workspace_bytes < need || (need && (!workspace || uintptr_t(workspace) % 16))) {
        set_error("mx_linear: needs a 16-byte aligned workspace of %zu bytes", need);
        return SCMX_ERR_WORKSPACE;
    }
    if (M && (!x || uintptr_t(x) % 2 || uintptr_t(nw) % 2 || (M > 1 && (ldx < K || ldx > INT64_MAX / 8 / M)) || (nw && K > 16384))) {
        set_error("mx_linear: need bf16 rows at least K apart, of up to 16384 values with a norm (M=%d K=%d ldx=%lld)", M, K,
                  (long long)ldx);
        return SCMX_ERR_ARG;
    }
    if (M == 0) return SCMX_OK;
    if (M == 1) ldx = K;
    if (in_one(M, N, K) && !nw) {   // (N is at most 2^24 then)
        FewArgs a{};
        static_cast<MxArgs&>(a) = MxArgs{nullptr, nullptr, wcodes, wscales, res, out, epi, M, N, K};
        a.rows = x;
        a.ldx = ldx;
        launch_few(a, (hipStream_t)stream);
        return check_launch("mx_linear");
    }
    uint8_t *codes = static_cast<uint8_t*>(workspace), *scales = codes + size_t(M) * (K / 2);
    if (int rc = scmx_mx_quantize(x, SCMX_MX_BF16, ldx, nw, eps, codes, scales, M, K, stream)) return rc;
    return scmx_mx_mm(codes, scales, wcodes, wscales, res, out, epi, M, N, K, stream);
}
