// Gradients of cross attention (rsfa_cross_bwd, declared in include/rsfa.h).
//
//   P = exp(s q k^T - lse),  dV = P^T dO,  dS = P (dO V^T - delta),  dQ = s dS K,  dK = s dS^T Q
//   delta = rowsum(dO o) - dlse
//
// Two kernels: dQ, whose workgroups hold a block of rows, form its delta and pass over the keys; then dK and dV, whose
// workgroups hold a block of keys and pass over the rows of their key head (all query heads of its group, so
// shared heads need no second sum).  Both form S and dO V^T, which makes seven matrix products where
// one kernel would have five, but every sum has one owner and one order: no atomics, the same bits in each call,
// and no traffic for dQ's partial sums, which one kernel would add up in memory once per key block.
// Where blocks are too few for the chip each pass is cut into parts, which sum_parts_kernel adds up.
//
// P and dS are rounded to the type for the products with rows (half a step of each, as the matrix unit takes 16-bit
// operands at sixteen times the rate of 32-bit ones); all else is in 32 bits.  float16 ends at 2^-14 and at 2^16, where
// gradients are often smaller or larger: P is scaled by 2^12 there, and dS by 2^k with a k for which it stays below 2^13 (so that
// there is room for weights above 1, as the roundings of scores of some millions may give).  As P <= 1 and
// |dO v| <= |dO| |v| (2-norms), |dS| of a key (dK) is at most |v| times the largest |dO| of the key head's rows plus
// their largest |delta|, which the dQ kernel leaves per 32 rows.  For a row (dQ) the largest |v| is not known ahead, but P |v| is about
// |o| at most, unless large values cancel in o: k goes by |dO| |o| + |delta|, with room for 2^SPARE times as much; where that was not
// enough the sums are not finite, and the workgroup finds the largest |v| and passes over its keys again.  2^k goes into the
// exponent and out at the end.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/rsfa.h"
#include "cross.hpp"

using namespace rsfa;

namespace {

constexpr float LOG2E = 1.4426950408889634f;
// Scores are multiplied by c = |sm_scale| * log2 e within the exponential; with a smaller c than this the part of lse / c
// that the number of keys makes up would overflow, and no weight is another but for scores q k above 2^100.
constexpr float LEAST_C = 7.523163845262640e-37f;  // 2^-120
constexpr int ROWS = 64;  // rows are padded to whole tiles of 64 in the statistics

struct BwdParams {
    const void *q, *k, *v, *o, *go;
    const float *lse, *glse;
    void *gq, *gk, *gv;
    int64_t q_st[3], k_st[3], v_st[3], o_st[3], go_st[3], gq_st[3], gk_st[3], gv_st[3];  // elements, of (Z, heads, rows)
    const int32_t* lengths;
    int32_t z, heads, key_heads, group, t, n;
    int32_t tp;        // t in whole tiles
    int32_t blocks;    // blocks of a key head (dK, dV) or of a query head (dQ)
    int32_t splits;    // parts of the pass
    float c, scale;
    uint32_t neg;      // sign of sm_scale, as a mask for a pair of values
    float *nl, *nd;    // [Z * heads][tp]: -lse / (c ln 2), -delta; rows past t: -inf, 0
    float2* top;       // float16: [Z * heads][tp / 32]: largest |dO| and |delta| of 32 rows
    float* part[2];    // splits > 1: [splits][rows][D] of dK and dV, or of dQ
};

__device__ __forceinline__ int keys_of(const BwdParams& p, int z) {
    return __builtin_amdgcn_readfirstlane(p.lengths ? max(0, min(p.lengths[z], p.n)) : p.n);
}

// One wave's direct load of 64 dwords into LDS (dma16's smaller sibling; see there for the s_nop).
__device__ __forceinline__ void dma4(const void* sbase, uint32_t voff_bytes, uint32_t lds_addr) {
    asm volatile("s_nop 4\n\tglobal_load_lds_dword %0, %1"
                 :
                 : "v"(voff_bytes), "s"(sbase), "{m0}"(lds_addr)
                 : "memory");
}

// The greatest k for which 2^k x stays below 2^13, within -100 .. 40, where P 2^k and its sums are far from the ends of 32 bits.
__device__ __forceinline__ float room(float x) {
    const int e = (int)(__float_as_uint(x) >> 23 & 255) - 127;
    return (float)max(-100, min(12 - e, 40));
}

constexpr float P_ROOM = 12.0f;  // of P itself
constexpr float SPARE = 6.0f;

template <class X8, int N>
__device__ __forceinline__ float sum_of_squares(const X8 (&x)[N]) {
    float sum = 0.0f;
#pragma unroll
    for (int s = 0; s < N; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = __builtin_fmaf((float)x[s][e], (float)x[s][e], sum);
    return sum;
}

// Tiles of rows in LDS have the forward kernel's layout (fa_fwd_kernel.hpp): 16-row blocks of planes of 32 columns,
// read as rows (A operand of S = Q K^T) and as transposes (A operand of dV^T = dO^T P) without bank conflicts.
struct Lane {
    int lane, hh, l32, l16;
    uint32_t koff[2], voff[2];
    int ld_row, ld_col;
    template <int D>
    __device__ __forceinline__ void set(int tid) {
        constexpr int BLK = 32 * D;
        lane = tid & 63, hh = lane >> 5, l32 = lane & 31, l16 = lane & 15;
#pragma unroll
        for (int e = 0; e < 2; ++e) koff[e] = (l32 >> 4) * BLK + l16 * 64 + ((2 * e + hh) ^ row_swz(l16)) * 16;
        const int vcc = 2 * ((lane >> 4) & 1) + ((l16 >> 1) & 1);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int r = 8 * u + 4 * hh + (l16 >> 2);
            voff[u] = r * 64 + (vcc ^ row_swz(r)) * 16 + 8 * (l16 & 1);
        }
        ld_row = lane >> 2, ld_col = ((lane & 3) ^ row_swz(ld_row)) * 8;
    }
};

// acc += A B over the D values of a row: A 32 rows of a tile in LDS, B in registers.
template <class T, int D>
__device__ __forceinline__ void rows_product(const RSFA_LDS char* tile, const Lane& w, const typename T::x8 (&b)[D / 16], f32x16& acc) {
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
        const typename T::x8 a = *(const RSFA_LDS typename T::x8*)(tile + w.koff[s & 1] + (s >> 1) * 1024);
        acc = T::mfma(a, b[s], acc);
    }
}

// acc[d] += A B over 32 rows of a tile: A the transpose of the tile's columns 32 d .., B in registers.
template <class T, int D>
__device__ __forceinline__ void columns_product(const RSFA_LDS char* tile, const Lane& w, const typename T::x8 (&b)[2], f32x16 (&acc)[D / 32]) {
    typedef typename T::x8 x8;
    constexpr int BLK = 32 * D;
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
            const RSFA_LDS char* const at = tile + h2 * BLK + d * 1024;
            const i32x2 lo = __builtin_bit_cast(i32x2, T::tr_read(at + w.voff[0]));
            const i32x2 hi = __builtin_bit_cast(i32x2, T::tr_read(at + w.voff[1]));
            acc[d] = T::mfma(__builtin_bit_cast(x8, (i32x4){lo[0], lo[1], hi[0], hi[1]}), b[h2], acc[d]);
        }
}

template <class T>
__device__ __forceinline__ void pack(const f32x16& x, typename T::x8 (&b)[2]) {
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const typename T::x2 pr = T::cvt2(x[8 * h2 + 2 * i], x[8 * h2 + 2 * i + 1]);
            b[h2][2 * i] = pr[0], b[h2][2 * i + 1] = pr[1];
        }
}

// A wave's 32 rows from `base` on into LDS of its own (rows behind the last of `left` repeat it), by direct loads of 16 rows x 64 bytes.
template <int D, class E>
__device__ __forceinline__ void load_rows(const E* base, int64_t st, int left, const Lane& w, uint32_t to) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int r0 = min(16 * b, left - 1);
        const uint32_t off = (uint32_t)(((min(r0 + w.ld_row, left - 1) - r0) * st + w.ld_col) * 2);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) dma16(base + r0 * st + 32 * c, off, to + b * (32 * D) + c * 1024);
    }
}

// Those rows as operands: lane l has row l % 32, values 16 s + 8 (l / 32) ...
template <class T, int D>
__device__ __forceinline__ void fragments(const RSFA_LDS char* at, const Lane& w, typename T::x8 (&f)[D / 16]) {
#pragma unroll
    for (int s = 0; s < D / 16; ++s) f[s] = *(const RSFA_LDS typename T::x8*)(at + w.koff[s & 1] + (s >> 1) * 1024);
}

// The 32 rows of a wave's transposed accumulator (lane l holds row l % 32, values 32 d + 8 a + 4 (l / 32) + e), times f, to
// memory, through LDS of its own: stored from the accumulator, every instruction would write 32 rows x 16 bytes, at 64 cycles
// of the address unit each; so a row's chunks of 16 bytes lie side by side.  Rows from `left` on are not written.
template <class T, int D>
__device__ __forceinline__ void store_rows(typename T::elem* dst, int64_t st, int left, const f32x16 (&acc)[D / 32], float f,
                                           const Lane& w, RSFA_LDS char* at) {
    typedef typename T::x8 x8;
    constexpr int COLS = D == 256 ? 128 : D;  // at once (all of D = 256 would not fit the wave's share)
    constexpr int PITCH = 2 * COLS + 16, CH = COLS / 8, EACH = 64 / CH;
    const int r0 = w.lane / CH, c = w.lane % CH;
#pragma unroll
    for (int part = 0; part < D / COLS; ++part) {
#pragma unroll
        for (int d = 0; d < COLS / 32; ++d)
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                typename T::x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (typename T::elem)(acc[part * (COLS / 32) + d][4 * a + e] * f);
                *(RSFA_LDS typename T::x4*)(at + w.l32 * PITCH + (32 * d + 8 * a + 4 * w.hh) * 2) = v;
            }
#pragma unroll
        for (int i = 0; i < 32 / EACH; ++i) {
            const int r = i * EACH + r0;
            const x8 v = *(const RSFA_LDS x8*)(at + r * PITCH + c * 16);
            if (r < left) *(x8*)(dst + r * st + part * COLS + 8 * c) = v;
        }
    }
}

template <int D>
__device__ __forceinline__ void store_part(float* dst, const f32x16 (&acc)[D / 32], float f, int hh) {
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int a = 0; a < 4; ++a)
            *(float4*)(dst + 32 * d + 8 * a + 4 * hh) = make_float4(acc[d][4 * a] * f, acc[d][4 * a + 1] * f, acc[d][4 * a + 2] * f, acc[d][4 * a + 3] * f);
}

// dK and dV of 128 keys, 32 of each wave, held transposed (dK^T = Q^T dS, dV^T = dO^T P): with keys in the lanes S
// and dS leave the matrix unit as the operands that the next products take.  K and V of the wave stay in registers;
// tiles of rows of Q and dO pass through LDS, two buffers.
// Bound by the matrix unit at D = 128: 8 x 32 heads of 2048 rows, 4096 keys of 8, bf16, 1684 us, 1306 TFLOP/s of its four products, as many
// as a large library product reaches; at D = 64 the vector unit, with an exponential, two products and half a conversion a score,
// has more to do than the matrix unit: 16 x 16 heads of 447 rows, 1531 keys, 850 TFLOP/s (float16, whose two scales are one more
// product a score, 108 us where one scale took 104).
template <int D>
struct Bwd {
    static constexpr int TILE_ROWS = D == 256 ? 32 : 64;
    static constexpr int DKV_OCC = D == 256 ? 1 : D == 32 ? 4 : D == 64 ? 3 : 2;  // waves of a SIMD
    static constexpr int DQ_OCC = D == 256 ? 1 : D <= 64 ? 4 : 2;
};

template <class T, int D>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(Bwd<D>::DKV_OCC, Bwd<D>::DKV_OCC)))
cross_dkv_kernel(BwdParams p) {
    typedef typename T::x8 x8;
    typedef typename T::elem elem;
    constexpr int QB = Bwd<D>::TILE_ROWS, BLK = 32 * D, TILE = QB * D * 2, STATS = 512, BUF = 2 * TILE + STATS;
    constexpr int TWO = QB == 64 ? 64 * D : 0;  // where a wave's second 32 rows lie in the LDS of its prologue
    constexpr int DT = D / 32, KST = D / 16;
    constexpr bool F16 = std::is_same<T, TypeF16>::value;
    __shared__ __attribute__((aligned(1024))) char smem_raw[2 * BUF];
    RSFA_LDS char* const smem = (RSFA_LDS char*)smem_raw;
    const uint32_t smem_addr = (uint32_t)(uintptr_t)smem;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Lane w;
    w.set<D>(threadIdx.x);
    int kh, block;
    head_block(p.z * p.key_heads, p.blocks, kh, block);
    const int z = kh / p.key_heads, h = kh - z * p.key_heads;
    const int nk = keys_of(p, z);
    const int key = block * 128 + wave * 32 + w.l32;

    const int tiles = (p.t + QB - 1) / QB, all = tiles * p.group;
    const int each = (all + p.splits - 1) / p.splits;
    int i = min((int)blockIdx.y * each, all);
    const int end = block * 128 < nk ? min(i + each, all) : i;  // (no key: no pass)
    const bool mine = i < end && block * 128 + wave * 32 < nk;  // the wave has work
    const int first = block * 128 + wave * 32;  // the wave's first key
    RSFA_LDS char* const own = smem + wave * TILE;
    x8 kf[KST], vf[KST];
    if (mine) {
        load_rows<D>((const elem*)p.k + z * p.k_st[0] + h * p.k_st[1] + first * p.k_st[2], p.k_st[2], nk - first, w, smem_addr + wave * TILE);
        if constexpr (TWO == 0) {  // (one after the other through the same place)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            fragments<T, D>(own, w, kf);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        load_rows<D>((const elem*)p.v + z * p.v_st[0] + h * p.v_st[1] + first * p.v_st[2], p.v_st[2], nk - first, w, smem_addr + wave * TILE + TWO);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if constexpr (TWO != 0) fragments<T, D>(own, w, kf);
        fragments<T, D>(own + TWO, w, vf);
#pragma unroll
        for (int s = 0; s < KST; ++s) kf[s] = __builtin_bit_cast(x8, __builtin_bit_cast(u32x4, kf[s]) ^ p.neg);
    }
    __syncthreads();  // (the tiles go where these rows were)
    float k2 = 0.0f, up = 1.0f;  // float16: of dS and, times up, of P
    if constexpr (F16) {
        const int n = p.group * (p.tp / 32);
        const float2* const top = p.top + (int64_t)kh * n;
        float go = 0.0f, delta = 0.0f;
        for (int j = w.lane; j < n; j += 64) go = fmaxf(go, top[j].x), delta = fmaxf(delta, top[j].y);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) go = fmaxf(go, __shfl_xor(go, d)), delta = fmaxf(delta, __shfl_xor(delta, d));
        float v2 = mine ? sum_of_squares(vf) : 0.0f;
        v2 += __shfl_xor(v2, 32);
        k2 = room(go * __builtin_sqrtf(v2) + delta);
        up = __builtin_amdgcn_exp2f(P_ROOM - k2);
    }
    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[d][r] = dv[d][r] = 0.0f;

    auto load = [&](int it, int buf) {
        const int g = it / tiles, row0 = (it - g * tiles) * QB;
        const int hq = h * p.group + g;
        const uint32_t dst = smem_addr + buf * BUF;
        const elem* qb = (const elem*)p.q + z * p.q_st[0] + hq * p.q_st[1];
        const elem* gb = (const elem*)p.go + z * p.go_st[0] + hq * p.go_st[1];
        const int last = p.t - 1;  // rows past it repeat it: their statistics make P 0 (and dO is hidden)
        auto rows = [&](const elem* base, int64_t st, int blk, uint32_t to) {
            const int r0 = min(row0 + 16 * blk, last);
            const uint32_t off = (uint32_t)(((min(r0 + w.ld_row, last) - r0) * st + w.ld_col) * 2);
            const elem* at = base + r0 * st;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) dma16(at + 32 * c, off, to + blk * BLK + c * 1024);
        };
        if constexpr (QB == 64) {
            rows(qb, p.q_st[2], wave, dst);
            rows(gb, p.go_st[2], wave, dst + TILE);
        } else if (wave < 2) {
            rows(qb, p.q_st[2], wave, dst);
        } else {
            rows(gb, p.go_st[2], wave - 2, dst + TILE);
        }
        // (32-row tiles load 64 dwords too: the statistics have room behind the last)
        if (wave < 2) {
            const int64_t at = (int64_t)(z * p.heads + hq) * p.tp + row0;
            dma4((wave ? p.nd : p.nl) + at, 4 * w.lane, dst + 2 * TILE + wave * 256);
        }
    };
    auto stats = [&](const RSFA_LDS char* at, f32x16& x) {
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const f32x4 v = *(const RSFA_LDS f32x4*)(at + (8 * a + 4 * w.hh) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * a + e] = v[e];
        }
    };

    int left = p.t - i % tiles * QB;  // rows from the tile's first on
    if (i < end) load(i, 0);
    for (int buf = 0; i < end; ++i, buf ^= 1, left = left > QB ? left - QB : p.t) {
        wait_loads_and_sync();
        if (i + 1 < end) load(i + 1, buf ^ 1);
        if (!mine) continue;
        const RSFA_LDS char* const qt = smem + buf * BUF;
        RSFA_LDS char* const gt = smem + buf * BUF + TILE;
        // (P of the rows that fill a tile up is 0, and 0 times an infinite dO would be NaN)
        if (__builtin_expect(left < QB, 0)) hide_rows<D, QB>(gt, left, w.lane);
#pragma unroll
        for (int st = 0; st < QB / 32; ++st) {
            f32x16 s, x;
            x8 b[2];
            stats(gt + TILE + st * 128, s);
            rows_product<T, D>(qt + st * 2 * BLK, w, kf, s);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(F16 ? __builtin_fmaf(s[r], p.c, k2) : s[r] * p.c);
            if constexpr (F16) {
                f32x16 x;
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] = s[r] * up;
                pack<T>(x, b);
            } else {
                pack<T>(s, b);
            }
            columns_product<T, D>(gt + st * 2 * BLK, w, b, dv);
            stats(gt + TILE + 256 + st * 128, x);
            rows_product<T, D>(gt + st * 2 * BLK, w, vf, x);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] *= x[r];
            pack<T>(s, b);
            columns_product<T, D>(qt + st * 2 * BLK, w, b, dk);
        }
    }
    const float unscale = __builtin_amdgcn_exp2f(-k2), unscale_p = F16 ? __builtin_amdgcn_exp2f(-P_ROOM) : 1.0f;
    if (p.splits > 1) {
        if (key >= nk) return;  // (the sum of the parts writes 0 there)
        const int64_t at = (((int64_t)blockIdx.y * p.z * p.key_heads + kh) * p.n + key) * D;
        if (p.gk) store_part<D>(p.part[0] + at, dk, unscale, w.hh);
        if (p.gv) store_part<D>(p.part[1] + at, dv, unscale_p, w.hh);
        return;
    }
    if (key >= nk) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) dk[d][r] = dv[d][r] = 0.0f;
    }
    __syncthreads();  // (every wave is done with the tiles)
    if (p.gk) store_rows<T, D>((elem*)p.gk + z * p.gk_st[0] + h * p.gk_st[1] + first * p.gk_st[2], p.gk_st[2], p.n - first, dk, p.scale * unscale, w, own);
    if (p.gv) store_rows<T, D>((elem*)p.gv + z * p.gv_st[0] + h * p.gv_st[1] + first * p.gv_st[2], p.gv_st[2], p.n - first, dv, unscale_p, w, own);
}

// dQ of 128 rows, 32 of each wave, held transposed (dQ^T = K^T dS^T), rows in the lanes: a row's
// statistics are one register each.  Q and dO of the wave stay in registers; tiles of K and V pass through LDS.
// Bound as dK and dV are: the same calls 1336 us, 1235 TFLOP/s of its three products, and 880 TFLOP/s; with few keys by memory:
// 8 x 8 heads of 4096 rows, 19 to 77 keys, D = 64, bf16 31 us, 4.4 TB/s of q, o, dO and dQ, float16, which forms |dO|, |o| and looks
// whether its sums are finite, 36, 3.7 TB/s.
template <class T, int D>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(Bwd<D>::DQ_OCC, Bwd<D>::DQ_OCC)))
cross_dq_kernel(BwdParams p) {
    typedef typename T::x8 x8;
    typedef typename T::elem elem;
    constexpr int KB = Bwd<D>::TILE_ROWS, BLK = 32 * D, TILE = KB * D * 2, BUF = 2 * TILE;
    constexpr int TWO = KB == 64 ? 64 * D : 0;  // where a wave's second 32 rows lie in the LDS of its prologue
    constexpr int DT = D / 32, KST = D / 16;
    constexpr bool F16 = std::is_same<T, TypeF16>::value;
    __shared__ __attribute__((aligned(1024))) char smem_raw[2 * BUF];
    RSFA_LDS char* const smem = (RSFA_LDS char*)smem_raw;
    const uint32_t smem_addr = (uint32_t)(uintptr_t)smem;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Lane w;
    w.set<D>(threadIdx.x);
    int kh, block;
    head_block(p.z * p.key_heads, p.blocks * p.group, kh, block);
    const int z = kh / p.key_heads, h = kh - z * p.key_heads;
    const int g = block / p.blocks, hq = h * p.group + g;
    block -= g * p.blocks;
    const int nk = keys_of(p, z);
    const int row = block * 128 + wave * 32 + w.l32;
    const bool mine = block * 128 + wave * 32 < p.t;

    const int all = (nk + KB - 1) / KB, each = (all + p.splits - 1) / p.splits;
    int i = min((int)blockIdx.y * each, all);
    const int end = p.gq ? min(i + each, all) : i;  // (without dQ the statistics are all there is to do)

    const int first = block * 128 + wave * 32;  // the wave's first row
    RSFA_LDS char* const own = smem + wave * TILE;
    x8 qf[KST], gf[KST];
    float l2 = 0.0f, nd = 0.0f, gl = 0.0f;
    float go = 0.0f, most = 0.0f;  // float16: |dO|; what |dO v| is taken to be at most
    if (mine) {
        const int64_t head = (int64_t)z * p.heads + hq;
        const int left = p.t - first;
        load_rows<D>((const elem*)p.q + z * p.q_st[0] + hq * p.q_st[1] + first * p.q_st[2], p.q_st[2], left, w, smem_addr + wave * TILE);
        if constexpr (TWO == 0) {  // (one after the other through the same place)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            fragments<T, D>(own, w, qf);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        load_rows<D>((const elem*)p.go + z * p.go_st[0] + hq * p.go_st[1] + first * p.go_st[2], p.go_st[2], left, w, smem_addr + wave * TILE + TWO);
        // o comes as the direct loads bring dO: lane l has chunk l % 4 (swizzled) of row l / 4 of a plane
        const elem* ob = (const elem*)p.o + z * p.o_st[0] + hq * p.o_st[1] + first * p.o_st[2] + w.ld_col;
        x8 o[2][D / 32];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int c = 0; c < D / 32; ++c) o[b][c] = *(const x8*)(ob + min(16 * b + w.ld_row, left - 1) * p.o_st[2] + 32 * c);
        const int row_c = min(row, p.t - 1);
        l2 = p.lse[head * p.t + row_c] * LOG2E;
        if (p.glse) gl = p.glse[head * p.t + row_c];
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if constexpr (TWO != 0) fragments<T, D>(own, w, qf);
        fragments<T, D>(own + TWO, w, gf);
#pragma unroll
        for (int s = 0; s < KST; ++s) qf[s] = __builtin_bit_cast(x8, __builtin_bit_cast(u32x4, qf[s]) ^ p.neg);
        float sum[2] = {0.0f, 0.0f}, o2[2] = {0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                const x8 gr = *(const RSFA_LDS x8*)(own + TWO + b * BLK + c * 1024 + w.lane * 16);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[b] = __builtin_fmaf((float)o[b][c][e], (float)gr[e], sum[b]);
            }
            sum[b] += __shfl_xor(sum[b], 1);
            sum[b] += __shfl_xor(sum[b], 2);
            if constexpr (F16) {
                o2[b] = sum_of_squares(o[b]);
                o2[b] += __shfl_xor(o2[b], 1);
                o2[b] += __shfl_xor(o2[b], 2);
            }
        }
        const float s0 = __shfl(sum[0], 4 * w.l16), s1 = __shfl(sum[1], 4 * w.l16);
        nd = gl - (w.l32 < 16 ? s0 : s1);
        if constexpr (F16) {
            go = sum_of_squares(gf);
            go = __builtin_sqrtf(go + __shfl_xor(go, 32));
            const float a = __shfl(o2[0], 4 * w.l16), b = __shfl(o2[1], 4 * w.l16);
            most = go * __builtin_sqrtf(w.l32 < 16 ? a : b);
        }
    }
    __syncthreads();  // (the tiles go where these rows were)
    f32x16 dq[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) dq[d][r] = 0.0f;

    const elem* const kb = (const elem*)p.k + z * p.k_st[0] + h * p.k_st[1];
    const elem* const vb = (const elem*)p.v + z * p.v_st[0] + h * p.v_st[1];
    auto load = [&](int it, int buf) {
        const int row0 = it * KB, last = nk - 1;
        const uint32_t dst = smem_addr + buf * BUF;
        auto rows = [&](const elem* base, int64_t st, int blk, uint32_t to) {
            const int r0 = min(row0 + 16 * blk, last);
            const uint32_t off = (uint32_t)(((min(r0 + w.ld_row, last) - r0) * st + w.ld_col) * 2);
            const elem* at = base + r0 * st;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) dma16(at + 32 * c, off, to + blk * BLK + c * 1024);
        };
        if constexpr (KB == 64) {
            rows(kb, p.k_st[2], wave, dst);
            rows(vb, p.v_st[2], wave, dst + TILE);
        } else if (wave < 2) {
            rows(kb, p.k_st[2], wave, dst);
        } else {
            rows(vb, p.v_st[2], wave - 2, dst + TILE);
        }
    };
    // S^T and (dO V^T)^T of 32 keys of tile `it`
    auto scores = [&](int it, int st, int buf, f32x16& s, f32x16& x) {
        const RSFA_LDS char* const kt = smem + buf * BUF;
        rows_product<T, D>(kt + st * 2 * BLK, w, qf, s);
        rows_product<T, D>(kt + TILE + st * 2 * BLK, w, gf, x);
        const int left = nk - it * KB - 32 * st - 4 * w.hh;  // keys of the sub-tile, from the lane's first on
        if (it * KB + 32 * st + 32 > nk) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (8 * (r / 4) + r % 4 >= left) s[r] = -INFINITY;
        }
    };
    // With few keys o is large and its rounding, in delta, would be as large as that of dS (8 keys, bfloat16: an error of dQ
    // against 64 bits of 0.0026 relative to it, 0.0024 without, 0.0017 being its own rounding): delta is then rowsum(P (dO V^T)).
    const bool once = all == 1 && i == 0;
    if (once) {
        load(0, 0);
        wait_loads_and_sync();
        if (mine) {
            float sum = 0.0f;
            most = 0.0f;
#pragma unroll
            for (int st = 0; st < KB / 32; ++st) {
                f32x16 s = {}, x = {};
                scores(0, st, 0, s, x);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    sum = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(s[r], p.c, -l2)), x[r], sum);
                    if (F16) most = fmaxf(most, __builtin_fabsf(x[r]));
                }
            }
            sum += __shfl_xor(sum, 32);
            nd = gl - sum;
            most = fmaxf(most, __shfl_xor(most, 32));
        }
    }
    // for dK and dV: rows behind the last have weights of 0
    if (blockIdx.y == 0 && w.hh == 0 && row < p.tp) {
        const int64_t at = ((int64_t)z * p.heads + hq) * p.tp + row;
        p.nl[at] = row < p.t ? -l2 / p.c : -INFINITY;
        p.nd[at] = row < p.t ? nd : 0.0f;
    }
    if constexpr (F16) {
        if (blockIdx.y == 0) {
            float a = go, b = __builtin_fabsf(nd);  // (0 for waves behind the last row)
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) a = fmaxf(a, __shfl_xor(a, d)), b = fmaxf(b, __shfl_xor(b, d));
            if (w.lane == 0 && first < p.tp) p.top[((int64_t)z * p.heads + hq) * (p.tp / 32) + first / 32] = make_float2(a, b);
        }
    }
    if (!p.gq) return;
    // -delta is what the products dO V^T start from where there is room for it: 16 registers instead of an addition a score (bf16,
    // eight sequences of 1500 keys, 1000 rows of 16 heads, D = 32 37.5 -> 35.0 us; four of 3000 keys, D = 128 95.5 -> 93.5; at D = 256
    // no difference.  D = 64 has no room with four waves a SIMD: float16, 64 heads of 4096 rows, 77 keys 32.2 -> 37.4)
    constexpr bool START = D == 32 || D == 128;
    f32x16 start = {};
    if constexpr (START) {
#pragma unroll
        for (int r = 0; r < 16; ++r) start[r] = nd;
        asm volatile("" : "+v"(start));  // (kept, and not formed again for each tile)
    }
    if (i < end && !once) load(i, 0);
    float k2 = 0.0f;  // float16: dS is scaled by 2^k2
    bool again = false;
    if constexpr (F16) {
        k2 = room(most + __builtin_fabsf(nd)) - (once ? 0.0f : SPARE);
        l2 -= k2;
    }
    for (const int begin = i;; i = begin) {
        for (int buf = 0; i < end; ++i, buf ^= 1) {
            wait_loads_and_sync();
            if (i + 1 < end) load(i + 1, buf ^ 1);
            if (!mine) continue;
            const RSFA_LDS char* const kt = smem + buf * BUF;
#pragma unroll
            for (int st = 0; st < KB / 32; ++st) {
                f32x16 s = {}, x = start;
                scores(i, st, buf, s, x);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], p.c, -l2)) * (START ? x[r] : x[r] + nd);
                x8 b[2];
                pack<T>(s, b);
                columns_product<T, D>(kt + st * 2 * BLK, w, b, dq);
            }
        }
        if constexpr (!F16) break;
        if (once || again) break;
        float test = 0.0f;  // NaN where a sum is not finite
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) test = __builtin_fmaf(dq[d][r], 0.0f, test);
        const bool over = __any(test != 0.0f);
        __shared__ float found[4];
        if (w.lane == 0) found[wave] = over ? 1.0f : 0.0f;
        __syncthreads();
        again = found[0] + found[1] + found[2] + found[3] != 0.0f;
        if (!again) break;
        constexpr int G = D / 8;  // lanes of a key
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));  // (nothing of this is formed ahead of the loop)
        float v2 = 0.0f;
        for (int64_t key = (int64_t)begin * KB + tid / G, last = min((int64_t)end * KB, (int64_t)nk); key < last; key += 256 / G) {
            const x8 v[1] = {*(const x8*)(vb + key * p.v_st[2] + 8 * (tid % G))};
            float sum = sum_of_squares(v);
#pragma unroll
            for (int d = 1; d < G; d <<= 1) sum += __shfl_xor(sum, d);
            v2 = fmaxf(v2, sum);
        }
#pragma unroll
        for (int d = G; d < 64; d <<= 1) v2 = fmaxf(v2, __shfl_xor(v2, d));
        __syncthreads();
        if (w.lane == 0) found[wave] = v2;
        __syncthreads();
        v2 = fmaxf(fmaxf(found[0], found[1]), fmaxf(found[2], found[3]));
        __syncthreads();
        l2 += k2;
        k2 = room(go * __builtin_sqrtf(v2) + __builtin_fabsf(nd));
        l2 -= k2;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) dq[d][r] = 0.0f;
        load(begin, 0);
    }
    if (p.splits > 1) {
        if (row >= p.t) return;
        const int64_t rows = (int64_t)p.z * p.heads * p.t;
        store_part<D>(p.part[0] + (blockIdx.y * rows + ((int64_t)z * p.heads + hq) * p.t + row) * D, dq, __builtin_amdgcn_exp2f(-k2), w.hh);
        return;
    }
    if (!F16 || once || again) __syncthreads();  // (every wave is done with the tiles)
    store_rows<T, D>((elem*)p.gq + z * p.gq_st[0] + hq * p.gq_st[1] + first * p.gq_st[2], p.gq_st[2], p.t - first, dq, p.scale * __builtin_amdgcn_exp2f(-k2), w, own);
}

// Sums of parts: D / 4 lanes a row; rows past their sequence's length (dK, dV) become 0.  Bound by the latency of the launch
// and of the loads, four under way together: eight parts of 64 heads' 77 rows, D = 64, both gradients 4.1 us.
struct SumParams {
    const float* part;
    void* out;
    int64_t st[3];
    const int32_t* lengths;  // or null
    int32_t heads, n, splits;
    int64_t rows;            // Z * heads * n
    float f;
};

template <class T, int D>
__global__ void __launch_bounds__(256) sum_parts_kernel(SumParams a, SumParams b) {
    typedef typename T::elem elem;
    const SumParams& p = blockIdx.y ? b : a;
    constexpr int G = D / 4;
    const int lane = threadIdx.x % G;
    const int64_t id = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (id >= p.rows) return;
    const int64_t zh = id / p.n;
    const int row = (int)(id - zh * p.n), z = (int)(zh / p.heads), h = (int)(zh - (int64_t)z * p.heads);
    f32x4 sum = {0, 0, 0, 0};
    if (!p.lengths || row < p.lengths[z]) {
#pragma unroll 4
        for (int s = 0; s < p.splits; ++s) sum += *(const f32x4*)(p.part + (s * p.rows + id) * D + 4 * lane);
    }
    typename T::x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (elem)(sum[i] * p.f);
    *(typename T::x4*)((elem*)p.out + z * p.st[0] + h * p.st[1] + row * p.st[2] + 4 * lane) = v;
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
struct Functions {
    const void *dkv, *dq, *sum;
};

template <class T>
Functions functions(int64_t d) {
    switch (d) {
        case 32: return {(const void*)&cross_dkv_kernel<T, 32>, (const void*)&cross_dq_kernel<T, 32>, (const void*)&sum_parts_kernel<T, 32>};
        case 64: return {(const void*)&cross_dkv_kernel<T, 64>, (const void*)&cross_dq_kernel<T, 64>, (const void*)&sum_parts_kernel<T, 64>};
        case 128: return {(const void*)&cross_dkv_kernel<T, 128>, (const void*)&cross_dq_kernel<T, 128>, (const void*)&sum_parts_kernel<T, 128>};
        default: return {(const void*)&cross_dkv_kernel<T, 256>, (const void*)&cross_dq_kernel<T, 256>, (const void*)&sum_parts_kernel<T, 256>};
    }
}

struct Plan {
    int64_t tp, key_blocks, row_blocks;
    int dkv_splits, dq_splits;
    uint64_t nl, nd, top, dkv[2], dq, bytes;
};

Plan make_plan(const rsfa_cross_bwd_args* a) {
    Plan p{};
    const int64_t d = a->head_dim, group = a->heads / a->key_heads, kh = a->z * a->key_heads, qh = a->z * a->heads;
    const int64_t tile = d == 256 ? 32 : 64, full = (int64_t)cross_cus() * (d == 256 ? 1 : d == 32 ? 4 : 2);
    p.tp = (a->t + ROWS - 1) / ROWS * ROWS;
    p.key_blocks = (a->n + 127) / 128;
    p.row_blocks = (a->t + 127) / 128;
    auto parts = [&](int64_t blocks, int64_t tiles) {
        return (int)std::max<int64_t>(1, std::min<int64_t>({full / blocks, tiles / 4, 64}));
    };
    p.dkv_splits = parts(kh * p.key_blocks, group * ((a->t + tile - 1) / tile));
    p.dq_splits = parts(qh * p.row_blocks, (a->n + tile - 1) / tile);
    uint64_t at = 0;
    auto take = [&](uint64_t n) {
        const uint64_t here = at;
        at += (n + 255) / 256 * 256;
        return here;
    };
    p.nl = take((uint64_t)qh * p.tp * 4 + 256);
    p.nd = take((uint64_t)qh * p.tp * 4 + 256);
    if (a->dtype == RSFA_DTYPE_F16) p.top = take((uint64_t)qh * p.tp / 32 * 8);
    if (p.dkv_splits > 1)
        for (int i = 0; i < 2; ++i) p.dkv[i] = take((uint64_t)p.dkv_splits * kh * a->n * d * 4);
    if (p.dq_splits > 1) p.dq = take((uint64_t)p.dq_splits * qh * a->t * d * 4);
    p.bytes = at;
    return p;
}

int check(const rsfa_cross_bwd_args* a) {
    if (!a) return RSFA_E_NULL;
    if (a->struct_size != sizeof(rsfa_cross_bwd_args)) return RSFA_E_ABI;
    return cross_check(a->dtype, a->z, a->heads, a->key_heads, a->t, a->n, a->head_dim);
}

}  // namespace

extern "C" {

uint64_t rsfa_cross_bwd_workspace_bytes(const rsfa_cross_bwd_args* a) { return check(a) == RSFA_OK ? make_plan(a).bytes : 0; }

int rsfa_cross_bwd(const rsfa_cross_bwd_args* a, void* stream) {
    int st = check(a);
    if (st != RSFA_OK) return st;
    if (!a->q || !a->k || !a->v || !a->o || !a->lse || !a->grad_o) return RSFA_E_NULL;
    struct {
        const void* at;
        const int64_t* st;
    } rows[] = {{a->q, a->q_stride}, {a->k, a->k_stride}, {a->v, a->v_stride}, {a->o, a->o_stride}, {a->grad_o, a->grad_o_stride},
                {a->grad_q, a->grad_q_stride}, {a->grad_k, a->grad_k_stride}, {a->grad_v, a->grad_v_stride}};
    for (auto& r : rows)
        if (r.at && (st = cross_check_rows(r.at, r.st)) != RSFA_OK) return st;
    if (((uintptr_t)a->lse | (uintptr_t)a->grad_lse | (uintptr_t)a->lengths) & 3) return RSFA_E_ALIGN;
    const Plan plan = make_plan(a);
    if (!a->workspace || a->workspace_bytes < plan.bytes) return RSFA_E_WORKSPACE;
    if ((uintptr_t)a->workspace & 15) return RSFA_E_ALIGN;
    char* const ws = (char*)a->workspace;
    BwdParams p{};
    p.q = a->q, p.k = a->k, p.v = a->v, p.o = a->o, p.go = a->grad_o, p.lse = a->lse, p.glse = a->grad_lse;
    p.gq = a->grad_q, p.gk = a->grad_k, p.gv = a->grad_v;
    for (int i = 0; i < 3; ++i) {
        p.q_st[i] = a->q_stride[i], p.k_st[i] = a->k_stride[i], p.v_st[i] = a->v_stride[i], p.o_st[i] = a->o_stride[i];
        p.go_st[i] = a->grad_o_stride[i], p.gq_st[i] = a->grad_q_stride[i], p.gk_st[i] = a->grad_k_stride[i], p.gv_st[i] = a->grad_v_stride[i];
    }
    p.lengths = a->lengths;
    p.z = (int32_t)a->z, p.heads = (int32_t)a->heads, p.key_heads = (int32_t)a->key_heads, p.group = p.heads / p.key_heads;
    p.t = (int32_t)a->t, p.n = (int32_t)a->n, p.tp = (int32_t)plan.tp;
    p.scale = a->sm_scale;
    p.c = std::max(std::fabs(a->sm_scale) * LOG2E, LEAST_C);
    p.neg = a->sm_scale < 0.0f ? 0x80008000u : 0u;
    p.nl = (float*)(ws + plan.nl), p.nd = (float*)(ws + plan.nd), p.top = (float2*)(ws + plan.top);
    const int64_t d = a->head_dim, kh = a->z * a->key_heads, qh = a->z * a->heads;
    const Functions fn = a->dtype == RSFA_DTYPE_BF16 ? functions<TypeBF16>(d) : functions<TypeF16>(d);
    const int64_t dkv_blocks = kh * plan.key_blocks, dq_blocks = qh * plan.row_blocks;
    const int64_t per = 1024 / d, sum_k = (kh * a->n + per - 1) / per, sum_q = (qh * a->t + per - 1) / per;
    if (std::max({dkv_blocks, dq_blocks, sum_k, sum_q}) > 0x7fffffff) return RSFA_E_CROSS;
    auto launch = [&](const void* f, int64_t x, int y, void** args) {
        return hipLaunchKernel(f, dim3((unsigned)x, (unsigned)y), dim3(256), args, 0, (hipStream_t)stream) == hipSuccess;
    };
    void* args[] = {&p};
    p.blocks = (int32_t)plan.row_blocks, p.splits = p.gq ? plan.dq_splits : 1;
    p.part[0] = (float*)(ws + plan.dq);
    if (!launch(fn.dq, dq_blocks, p.splits, args)) return RSFA_E_LAUNCH;
    if (p.splits > 1) {
        SumParams s[2] = {{p.part[0], p.gq, {p.gq_st[0], p.gq_st[1], p.gq_st[2]}, nullptr, p.heads, p.t, p.splits, qh * a->t, p.scale}, {}};
        void* sum_args[] = {&s[0], &s[1]};
        if (!launch(fn.sum, sum_q, 1, sum_args)) return RSFA_E_LAUNCH;
    }
    if (!p.gk && !p.gv) return RSFA_OK;
    p.blocks = (int32_t)plan.key_blocks, p.splits = plan.dkv_splits;
    for (int i = 0; i < 2; ++i) p.part[i] = (float*)(ws + plan.dkv[i]);
    if (!launch(fn.dkv, dkv_blocks, p.splits, args)) return RSFA_E_LAUNCH;
    if (p.splits > 1) {
        SumParams s[2] = {};
        int n = 0;
        if (p.gk) s[n++] = {p.part[0], p.gk, {p.gk_st[0], p.gk_st[1], p.gk_st[2]}, p.lengths, p.key_heads, p.n, p.splits, kh * a->n, p.scale};
        if (p.gv) s[n++] = {p.part[1], p.gv, {p.gv_st[0], p.gv_st[1], p.gv_st[2]}, p.lengths, p.key_heads, p.n, p.splits, kh * a->n, 1.0f};
        void* sum_args[] = {&s[0], &s[1]};
        if (!launch(fn.sum, sum_k, n, sum_args)) return RSFA_E_LAUNCH;
    }
    return RSFA_OK;
}

}  // extern "C"
