// Cross attention, forward (rsfa_cross_fwd, declared in include/rsfa.h).
//
//   o = softmax(sm_scale q k^T) v,  q [Z, heads, T, D],  k, v [Z, key heads, N, D]
//
// Many query tokens run the forward kernel (fa_fwd_kernel.hpp, MODE_CROSS), a task being a block
// of one query head's tokens; with too few tasks for the chip each takes a part of the keys.  Few
// tokens run cross_few_kernel below, which packs the rows (tokens and query heads) that share a key
// head and always has the keys in parts.  Parts are added up by join_kernel.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "../../include/rsfa.h"
#include "cross.hpp"
#include "kernel_table.hpp"

using namespace rsfa;

namespace {

constexpr float LN2 = 0.6931471805599453f;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float SLACK = 8.0f;  // how far (log2 units) a score may pass the running maximum: weights stay below 2^8

struct FewParams {
    const void *q, *k, *v;
    void* o;
    float* lse;
    int64_t q_st[3], k_st[3], v_st[3], o_st[3];  // element strides of (Z, heads, rows)
    const int32_t* lengths;
    int32_t heads, key_heads, group, t, n, bh;   // bh = Z * key heads
    int32_t rows;                                // group * t: row = token * group + head of the group
    int32_t tiles;                               // row tiles of a key head
    int32_t splits;
    float c;                                     // |sm_scale| * log2 e
    uint32_t neg;                                // sign of sm_scale, as a mask for a pair of q's values
    float* part_o;                               // [splits][Z * heads * t][D] (splits > 1)
    float2* part_ml;                             // [splits][Z * heads * t]: maximum (log2 units), sum
};

// Few rows (NB blocks of 16): each wave of a workgroup takes every WAVES-th tile of 32 keys of its part,
// and they add up what they have at the end.  A wave's tiles go from memory straight into LDS of its own,
// two buffers, so that a tile is under way while one is computed with and no barrier is needed.  In LDS a tile
// has the layout of the forward kernel (fa_fwd_kernel.hpp), whose rows and transposes are read without bank conflicts:
//   S^T = K Q^T   (v_mfma 16x16x32) A: lane l has the key l % 16 and values 8 (l / 16) .. of a step of 32
//   O^T = V^T P^T  S^T leaves lane l the row l % 16 and keys 16 t + 4 (l / 16) + r; step k = 8 (l / 16) + 4 t + r takes
//                 them as they are, and A, two transposing reads a lane, has the same keys.
// Bound by memory: 4 D bytes a key, whatever the rows.  One token of 32 heads over 8192 keys of 8, D = 128, in 32 parts 8.4 us, 4.0
// TB/s (parts of 16 KB a wave: the launch and the first loads take half); one token of 32 sequences, 16 heads, 382 to 1531 keys, D = 64
// 34 us, 3.8 TB/s, 5.3 where all have 1531.
template <class T, int D, int NB>
__global__ void __launch_bounds__(64 * Few<D>::WAVES, Few<D>::OCC) cross_few_kernel(FewParams p) {
    typedef typename T::elem elem;
    typedef typename T::x8 x8;
    constexpr int WAVES = Few<D>::WAVES, KEYS = 32, STEP = KEYS * WAVES;
    constexpr int QS = D / 32, DT = D / 16;
    constexpr int BLK = 32 * D;          // bytes of 16 rows
    constexpr int TILE = KEYS * D * 2;   // bytes of a K or V tile
    constexpr int LOADS = TILE / 1024;   // direct loads of one
    constexpr int ROWS = 16 * NB, PITCH = D + 4;
    constexpr int BUFFERS = WAVES * 2 * 2 * TILE, SUMS = WAVES * ROWS * (PITCH * 4 + 8);
    __shared__ __attribute__((aligned(1024))) char smem_raw[BUFFERS > SUMS ? BUFFERS : SUMS];
    RSFA_LDS char* const smem = (RSFA_LDS char*)smem_raw;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    int bh, block;
    head_block(p.bh, p.tiles, bh, block);
    const int row0 = block * ROWS;
    const int z = bh / p.key_heads, h = bh - z * p.key_heads;
    const int len = __builtin_amdgcn_readfirstlane(p.lengths ? max(0, min(p.lengths[z], p.n)) : p.n);
    const int chunk = ((len + p.splits - 1) / p.splits + STEP - 1) / STEP * STEP;
    const int64_t start64 = (int64_t)chunk * blockIdx.y;
    const int start = (int)(start64 < len ? start64 : len);
    const int end = min(start + chunk, len);

    const elem* const kb = (const elem*)p.k + z * p.k_st[0] + h * p.k_st[1];
    const elem* const vb = (const elem*)p.v + z * p.v_st[0] + h * p.v_st[1];
    const uint32_t lds0 = (uint32_t)(uintptr_t)smem + wave * (4 * TILE);  // buffer b: K at 2 b TILE, V behind
    // lane i of a load fills chunk i % 4 of row i / 4 of a plane of 16 rows x 32 values
    const int ld_row = lane >> 2, ld_col = ((lane & 3) ^ row_swz(ld_row)) * 8;
    auto load = [&](int tile, int buf) {
        const uint32_t dst = lds0 + buf * (2 * TILE);
        const int last = len - 1 - tile;  // rows behind the last key repeat it (compute hides them)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int row = min(16 * b + ld_row, last);
            const uint32_t ko = (uint32_t)((row * p.k_st[2] + ld_col) * 2), vo = (uint32_t)((row * p.v_st[2] + ld_col) * 2);
            const elem *kt = kb + tile * p.k_st[2], *vt = vb + tile * p.v_st[2];
#pragma unroll
            for (int i = 0; i < D / 32; ++i) dma16(kt + 32 * i, ko, dst + b * BLK + i * 1024);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) dma16(vt + 32 * i, vo, dst + TILE + b * BLK + i * 1024);
        }
    };
    const int tiles = (end - start + KEYS - 1) / KEYS;
    const int turns = tiles > wave ? (tiles - wave + WAVES - 1) / WAVES : 0;

    // Q^T (ahead of the tiles: the wait for it would wait for them)
    x8 q[NB][QS];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int row = row0 + 16 * b + col;
        const int tok = row / p.group, head = row - tok * p.group;
        u32x4 w[QS] = {};
        if (row < p.rows) {
            const elem* src = (const elem*)p.q + z * p.q_st[0] + (int64_t)(h * p.group + head) * p.q_st[1] + tok * p.q_st[2] + 8 * grp;
#pragma unroll
            for (int i = 0; i < QS; ++i) w[i] = *(const u32x4*)(src + 32 * i);
        }
#pragma unroll
        for (int i = 0; i < QS; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[i][j] ^= p.neg;
            q[b][i] = __builtin_bit_cast(x8, w[i]);
        }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < QS; ++i) asm volatile("" : "+v"(q[b][i]));
    if (turns) load(start + KEYS * wave, 0);

    f32x4 acc[NB][DT];
    float m[NB], l[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        m[b] = NEVER;
        l[b] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[b][d] = (f32x4){0, 0, 0, 0};
    }
    const uint32_t koff = col * 64 + (grp ^ row_swz(col)) * 16;
    const int vrow = 4 * grp + (col >> 2);
    uint32_t voff[2];  // even and odd blocks of 16 values
#pragma unroll
    for (int e = 0; e < 2; ++e) voff[e] = vrow * 64 + ((2 * e + ((col >> 1) & 1)) ^ row_swz(vrow)) * 16 + 8 * (col & 1);

    auto compute = [&](int buf, int tile) {
        const RSFA_LDS char* const kt = smem + wave * (4 * TILE) + buf * (2 * TILE);
        RSFA_LDS char* const vt = smem + wave * (4 * TILE) + buf * (2 * TILE) + TILE;
        if (__builtin_expect(tile + KEYS > end, 0)) hide_rows<D, KEYS>(vt, end - tile, lane);
        f32x4 s[NB][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int b = 0; b < NB; ++b) s[b][t] = (f32x4){0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < QS; ++i) {
                const x8 a = *(const RSFA_LDS x8*)(kt + t * BLK + i * 1024 + koff);
#pragma unroll
                for (int b = 0; b < NB; ++b) s[b][t] = mfma16(a, q[b][i], s[b][t]);
            }
        }
        x8 pk[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = s[b][j / 4][j % 4] * p.c;
            if (__builtin_expect(tile + KEYS > end, 0)) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (tile + 16 * (j / 4) + 4 * grp + j % 4 >= end) x[j] = -INFINITY;
            }
            float top = x[0];
#pragma unroll
            for (int j = 1; j < 8; ++j) top = fmaxf(top, x[j]);
            if (__any(top > m[b] + SLACK)) {
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float now = fmaxf(m[b], top);
                const float f = __builtin_amdgcn_exp2f(m[b] - now);
                m[b] = now;
                l[b] *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[b][d] *= f;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_exp2f(x[j] - m[b]);
            l[b] += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
#pragma unroll
            for (int j = 0; j < 8; ++j) pk[b][j] = (elem)x[j];
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const RSFA_LDS char* const at = vt + (d / 2) * 1024 + voff[d & 1];
            const i32x2 lo = __builtin_bit_cast(i32x2, T::tr_read(at));
            const i32x2 hi = __builtin_bit_cast(i32x2, T::tr_read(at + BLK));
            const x8 a = __builtin_bit_cast(x8, (i32x4){lo[0], lo[1], hi[0], hi[1]});
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[b][d] = mfma16(a, pk[b], acc[b][d]);
        }
    };

    for (int i = 0; i < turns; ++i) {
        const int tile = start + KEYS * (wave + WAVES * i);
        // the other buffer's reads have all been used, as its products have been issued
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (i + 1 < turns) {
            load(tile + STEP, (i + 1) & 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LOADS) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        compute(i & 1, tile);
    }

#pragma unroll
    for (int b = 0; b < NB; ++b) {
        l[b] += __shfl_xor(l[b], 16);
        l[b] += __shfl_xor(l[b], 32);
    }
    // the waves add up what they have, through LDS: each leaves its sums, scaled to the rows' common
    // maximum, and every thread adds E values of a row
    constexpr int THREADS = 64 * WAVES, E = ROWS * D / THREADS;
    __syncthreads();  // (the tiles' LDS is used again)
    RSFA_LDS float2* const ml = (RSFA_LDS float2*)(smem + WAVES * ROWS * PITCH * 4);
    RSFA_LDS float* const part = (RSFA_LDS float*)smem;
    auto put = [&](RSFA_LDS float2* at, float2 v) { ((RSFA_LDS float*)at)[0] = v.x, ((RSFA_LDS float*)at)[1] = v.y; };
    auto get = [&](const RSFA_LDS float2* at) { return make_float2(((const RSFA_LDS float*)at)[0], ((const RSFA_LDS float*)at)[1]); };
#pragma unroll
    for (int b = 0; b < NB; ++b)
        if (grp == 0) put(ml + wave * ROWS + 16 * b + col, make_float2(m[b], l[b]));
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        float mm = NEVER;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) mm = fmaxf(mm, get(ml + k * ROWS + 16 * b + col).x);
        const float f = __builtin_amdgcn_exp2f(m[b] - mm);
        RSFA_LDS float* const at = part + (wave * ROWS + 16 * b + col) * PITCH + 4 * grp;
#pragma unroll
        for (int d = 0; d < DT; ++d) *(RSFA_LDS f32x4*)(at + 16 * d) = acc[b][d] * f;
    }
    __syncthreads();
    const int r = threadIdx.x / (D / E), d0 = threadIdx.x % (D / E) * E;
    const int row = row0 + r;
    if (row >= p.rows) return;
    float mm = NEVER, ll = 0.0f;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) mm = fmaxf(mm, get(ml + k * ROWS + r).x);
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
        const float2 v = get(ml + k * ROWS + r);
        ll += v.y * __builtin_amdgcn_exp2f(v.x - mm);
    }
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        sum[e] = 0.0f;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) sum[e] += part[(k * ROWS + r) * PITCH + d0 + e];
    }
    const int tok = row / p.group, head = row - tok * p.group;
    const int64_t hq = h * p.group + head;
    const int64_t out = (z * (int64_t)p.heads + hq) * p.t + tok;
    if (p.splits > 1) {
        const int64_t at = blockIdx.y * ((int64_t)p.bh * p.rows) + out;
        if (d0 == 0) p.part_ml[at] = make_float2(mm, ll);
#pragma unroll
        for (int e = 0; e < E; e += 2) *(float2*)(p.part_o + at * D + d0 + e) = make_float2(sum[e], sum[e + 1]);
        return;
    }
    const float inv = len == 0 ? 0.0f : 1.0f / ll;
    elem* const dst = (elem*)p.o + z * p.o_st[0] + hq * p.o_st[1] + tok * p.o_st[2] + d0;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        typename T::x2 v = {(elem)(sum[e] * inv), (elem)(sum[e + 1] * inv)};
        *(typename T::x2*)(dst + e) = v;
    }
    if (d0 == 0 && p.lse) p.lse[out] = len == 0 ? -INFINITY : (mm + __builtin_amdgcn_logf(ll)) * LN2;
}

// Sums of the rows' parts: D / 4 lanes hold a row, four values each, and `pp` such groups of a
// workgroup take every pp-th part of it, so that the loads of a row's parts do not wait for each other.  Bound by the latency of the
// launch and of two loads: 32 parts of 32 rows, D = 128 3.3 us.
struct JoinParams {
    const float* part_o;
    const float2* part_ml;
    void* o;
    float* lse;
    int64_t o_st[3];
    const int32_t* lengths;
    int32_t heads, t, splits, pp;
    int64_t rows;  // Z * heads * t
};

template <class T, int D>
__global__ void __launch_bounds__(256) cross_join_kernel(JoinParams p) {
    constexpr int G = D / 4, GROUPS = 256 / G;
    __shared__ f32x4 part[256];
    __shared__ float2 ml[GROUPS];
    const int lane = threadIdx.x % G, grp = threadIdx.x / G;
    const int64_t id = (int64_t)blockIdx.x * (GROUPS / p.pp) + grp / p.pp;
    float m = -INFINITY, l = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    auto add = [&](float2 v, f32x4 x) {
        const float now = fmaxf(m, v.x);
        const float f = m == now ? 1.0f : __builtin_amdgcn_exp2f(m - now), g = v.x == now ? 1.0f : __builtin_amdgcn_exp2f(v.x - now);
        m = now;
        l = l * f + v.y * g;
        o = o * f + x * g;
    };
    if (id < p.rows) {
        constexpr int U = 8;  // parts whose loads are under way together
        for (int s0 = grp % p.pp; s0 < p.splits; s0 += U * p.pp) {
            float2 v[U];
            f32x4 x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int s = min(s0 + u * p.pp, p.splits - 1);
                v[u] = p.part_ml[s * p.rows + id];
                x[u] = *(const f32x4*)(p.part_o + (s * p.rows + id) * D + 4 * lane);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s0 + u * p.pp < p.splits) add(v[u], x[u]);
        }
    }
    if (p.pp > 1) {
        part[threadIdx.x] = o;
        if (lane == 0) ml[grp] = make_float2(m, l);
        __syncthreads();
        if (grp % p.pp != 0) return;
        for (int i = 1; i < p.pp; ++i) add(ml[grp + i], part[threadIdx.x + i * G]);
    }
    if (id >= p.rows) return;
    const int64_t zh = id / p.t;
    const int tok = (int)(id - zh * p.t), z = (int)(zh / p.heads), hq = (int)(zh - (int64_t)z * p.heads);
    const bool none = p.lengths ? p.lengths[z] <= 0 : false;
    const float inv = none ? 0.0f : 1.0f / l;
    typedef typename T::elem elem;
    elem* const dst = (elem*)p.o + z * p.o_st[0] + hq * p.o_st[1] + tok * p.o_st[2] + 4 * lane;
    typename T::x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (elem)(o[i] * inv);
    *(typename T::x4*)dst = w;
    if (lane == 0 && p.lse) p.lse[id] = none ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * LN2;
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
struct Plan {
    bool few;
    int nb;                // few: blocks of 16 rows a workgroup
    int64_t tiles;         // few: row tiles of a key head
    const KernelEntry* e;  // many
    int splits;
    uint64_t part_o, part_ml, bytes;
};

template <class T, int D>
const void* few_fn(int nb) {
    if constexpr (D < 256)
        if (nb == 4) return (const void*)&cross_few_kernel<T, D, 4>;
    return nb == 1 ? (const void*)&cross_few_kernel<T, D, 1> : (const void*)&cross_few_kernel<T, D, 2>;
}

template <class T>
const void* few_fn(int64_t d, int nb) {
    return d == 32 ? few_fn<T, 32>(nb) : d == 64 ? few_fn<T, 64>(nb) : d == 128 ? few_fn<T, 128>(nb) : few_fn<T, 256>(nb);
}

template <class T>
const void* join_fn(int64_t d) {
    switch (d) {
        case 32: return (const void*)&cross_join_kernel<T, 32>;
        case 64: return (const void*)&cross_join_kernel<T, 64>;
        case 128: return (const void*)&cross_join_kernel<T, 128>;
        default: return (const void*)&cross_join_kernel<T, 256>;
    }
}

int few_waves(int64_t d) { return d == 256 ? Few<256>::WAVES : Few<128>::WAVES; }

// What a call takes is read off a model, in microseconds, of launches that pass `steps` tiles of keys; the least of
// all variants and numbers of parts runs.  Measured on an MI355X in bfloat16, states in turn so that none stays in the last-level cache:
//   few rows, 16, 32, 64 of them a workgroup: 8 key heads of 8192 keys, D = 128, 16 rows: 51, 68, 107 us, in 16 parts
//   13, 14, 16; 128 heads of 1531, D = 64: 64 tokens 19, 14, 18, 200 tokens 44, 32, 25, the forward kernel 27;
//   512 heads of 1500, D = 64: 64 tokens 66, 44, 40, 128 tokens 105, 68, 50, the forward kernel 45.
//   The forward kernel's 8 and 4 waves: 128 heads of 1024 tokens, 4096 keys, D = 128: 249, 280; 64 heads of 4096
//   tokens, D = 64: 77 keys 32, 23, 512 keys 52, 46; 16 heads of 200 tokens, 4096 keys, D = 256: 160, 133, in 16 parts 56, 29.
constexpr double START_US = 4.0, FEW_US = 1.0, JOIN_US = 3.5;
constexpr double READ_US = 1.0 / 5.3e6, PART_US = 1.0 / 4.0e6;  // a byte of keys; a byte of parts, each way
struct FewCost {
    int d, keys, per_cu;  // keys of a step (all waves), workgroups of a CU
    double step[3];       // 16, 32, 64 rows
};
constexpr FewCost few_costs[] = {{32, 128, 4, {0.38, 0.49, 0.82}}, {64, 128, 2, {0.65, 0.78, 1.13}},
                                 {128, 128, 1, {0.82, 1.00, 1.65}}, {256, 64, 1, {1.30, 1.60, 0.0}}};
struct ManyCost {
    int d, nw, bn, per_cu;
    double task, step, task_shared, step_shared;  // shared: with per_cu workgroups on the CU
    double full;                                  // factor of a filled launch, at the board's power limit
};
constexpr ManyCost many_costs[] = {{32, 4, 64, 4, 0.23, 0.61, 1.25, 0.83, 1.5},  {32, 4, 128, 3, 0.23, 1.10, 1.25, 1.50, 1.5},
                                   {64, 8, 128, 1, 3.03, 1.49, 3.03, 1.49, 1.5}, {64, 4, 64, 3, 1.07, 0.90, 3.60, 1.30, 1.0},
                                   {128, 8, 64, 1, 3.00, 1.34, 3.00, 1.34, 1.5}, {128, 4, 64, 2, 2.04, 1.15, 3.44, 1.48, 1.5},
                                   {256, 8, 32, 1, 4.00, 1.22, 4.00, 1.22, 1.5}, {256, 4, 32, 2, 3.00, 1.00, 4.50, 1.30, 1.5}};

Plan make_plan(const rsfa_cross_args* a) {
    Plan p{};
    const int cus = cross_cus();
    const int64_t d = a->head_dim, rows = a->heads / a->key_heads * a->t, bh = a->z * a->key_heads, all = a->z * a->heads * a->t;
    const double read = 2.0 * 2.0 * (double)bh * a->n * d * READ_US;
    double best = 0.0;
    auto take = [&](double us, int64_t workgroups, int splits, bool few, int nb, const KernelEntry* e) {
        // (some CUs alone do not draw all of the memory's rate; reading and computing overlap for the most part)
        const double bytes = read / (0.6 + 0.4 * std::min(1.0, (double)workgroups / cus));
        us = START_US + std::max(us, bytes) + 0.25 * std::min(us, bytes);
        if (splits > 1) us += JOIN_US + 2.0 * 4.0 * splits * (double)all * d * PART_US;
        if (best != 0.0 && us >= best) return;
        best = us;
        p.few = few, p.nb = nb, p.e = e, p.splits = splits;
    };
    const KernelList list = a->dtype == RSFA_DTYPE_BF16 ? kernels_cross_bf16() : kernels_cross_f16();
    for (int splits = 1; splits <= 64; splits *= 2) {
        if (splits > 1 && a->n < 128 * (int64_t)splits) break;  // (parts of whole steps)
        const int64_t keys = (a->n + splits - 1) / splits;
        for (const FewCost& c : few_costs) {
            if (c.d != d) continue;
            for (int i = 0; i < 3 && c.step[i] != 0.0; ++i) {
                const int nb = 1 << i;
                if (i && 8 * nb >= rows) break;
                const int64_t workgroups = bh * ((rows + 16 * nb - 1) / (16 * nb)) * splits;
                const double alone = FEW_US + c.step[i] * (double)((keys + c.keys - 1) / c.keys), per = (double)workgroups / cus;
                // a CU's second workgroup and those after it add less than half of the first's time
                const double shared = alone * (1.0 + 0.45 * (std::min<double>(std::max(per, 1.0), c.per_cu) - 1.0));
                take(shared * std::max(1.0, std::ceil(per / c.per_cu - 1e-9)), workgroups, splits, true, nb, nullptr);
            }
        }
        for (const ManyCost& c : many_costs) {
            if (c.d != d) continue;
            const int64_t tasks = a->z * a->heads * ((a->t + 32 * c.nw - 1) / (32 * c.nw)) * splits;
            const int64_t conc = std::max<int64_t>(1, std::min<int64_t>(c.per_cu, (tasks + cus - 1) / cus)), slots = cus * conc;
            const double w = c.per_cu > 1 ? (double)(conc - 1) / (c.per_cu - 1) : 0.0;
            const double task = c.task + w * (c.task_shared - c.task) + (c.step + w * (c.step_shared - c.step)) * (double)((keys + c.bn - 1) / c.bn);
            const double us = std::max(task * (double)((tasks + slots - 1) / slots), task * (double)tasks / (double)(cus * c.per_cu) * c.full);
            for (int i = 0; i < list.count; ++i)
                if (list.entries[i].d == d && list.entries[i].nw == c.nw && list.entries[i].bn == c.bn)
                    take(us, tasks, splits, false, 0, &list.entries[i]);
        }
    }
    p.tiles = p.few ? (rows + 16 * p.nb - 1) / (16 * p.nb) : 0;
    if (p.splits > 1) {
        p.part_ml = 0;
        p.part_o = ((uint64_t)p.splits * all * 8 + 255) / 256 * 256;
        p.bytes = p.part_o + (uint64_t)p.splits * all * d * 4;
    }
    return p;
}

int check(const rsfa_cross_args* a) {
    if (!a) return RSFA_E_NULL;
    if (a->struct_size != sizeof(rsfa_cross_args)) return RSFA_E_ABI;
    return cross_check(a->dtype, a->z, a->heads, a->key_heads, a->t, a->n, a->head_dim);
}

}  // namespace

extern "C" {

uint64_t rsfa_cross_fwd_workspace_bytes(const rsfa_cross_args* a) { return check(a) == RSFA_OK ? make_plan(a).bytes : 0; }

int rsfa_cross_fwd(const rsfa_cross_args* a, void* stream) {
    int st = check(a);
    if (st != RSFA_OK) return st;
    if (!a->q || !a->k || !a->v || !a->o) return RSFA_E_NULL;
    for (auto [ptr, strides] : {std::pair(a->q, a->q_stride), std::pair(a->k, a->k_stride), std::pair(a->v, a->v_stride),
                                std::pair((const void*)a->o, a->o_stride)})
        if ((st = cross_check_rows(ptr, strides)) != RSFA_OK) return st;
    if (((uintptr_t)a->lse | (uintptr_t)a->lengths) & 3) return RSFA_E_ALIGN;
    const Plan plan = make_plan(a);
    if (plan.bytes) {
        if (!a->workspace || a->workspace_bytes < plan.bytes) return RSFA_E_WORKSPACE;
        if ((uintptr_t)a->workspace & 15) return RSFA_E_ALIGN;
    }
    const bool bf16 = a->dtype == RSFA_DTYPE_BF16;
    // (a scale of 0 would make a hidden score -inf * 0; at FLT_MIN the others still have weights of 1)
    const float c = std::max(std::fabs(a->sm_scale) * LOG2E, FLT_MIN);
    float2* const part_ml = plan.bytes ? (float2*)((char*)a->workspace + plan.part_ml) : nullptr;
    float* const part_o = plan.bytes ? (float*)((char*)a->workspace + plan.part_o) : nullptr;
    if (plan.few) {
        FewParams p{};
        p.q = a->q, p.k = a->k, p.v = a->v, p.o = a->o, p.lse = a->lse;
        for (int i = 0; i < 3; ++i) p.q_st[i] = a->q_stride[i], p.k_st[i] = a->k_stride[i], p.v_st[i] = a->v_stride[i], p.o_st[i] = a->o_stride[i];
        p.lengths = a->lengths;
        p.heads = (int32_t)a->heads, p.key_heads = (int32_t)a->key_heads, p.group = (int32_t)(a->heads / a->key_heads);
        p.t = (int32_t)a->t, p.n = (int32_t)a->n, p.bh = (int32_t)(a->z * a->key_heads), p.rows = p.group * p.t;
        p.tiles = (int32_t)plan.tiles;
        p.splits = plan.splits, p.c = c, p.neg = a->sm_scale < 0.0f ? 0x80008000u : 0u;
        p.part_o = part_o, p.part_ml = part_ml;
        const int64_t grid = p.bh * plan.tiles;
        if (grid > 0x7fffffff) return RSFA_E_CROSS;
        void* args[] = {&p};
        const void* fn = bf16 ? few_fn<TypeBF16>(a->head_dim, plan.nb) : few_fn<TypeF16>(a->head_dim, plan.nb);
        if (hipLaunchKernel(fn, dim3((unsigned)grid, (unsigned)plan.splits), dim3(64 * few_waves(a->head_dim)), args, 0, (hipStream_t)stream) != hipSuccess)
            return RSFA_E_LAUNCH;
    } else {
        FwdParams p{};
        p.q = a->q, p.k = a->k, p.v = a->v, p.o = a->o, p.lse = a->lse;
        p.q_sz = a->q_stride[0], p.q_sh = a->q_stride[1], p.q_sm = a->q_stride[2];
        p.k_sz = a->k_stride[0], p.k_sh = a->k_stride[1], p.k_sn = a->k_stride[2];
        p.v_sz = a->v_stride[0], p.v_sh = a->v_stride[1], p.v_sn = a->v_stride[2];
        p.o_sz = a->o_stride[0], p.o_sh = a->o_stride[1], p.o_sm = a->o_stride[2];
        p.H = (int32_t)a->key_heads;
        p.num_heads = (int32_t)(a->z * a->key_heads);
        p.group = (int32_t)(a->heads / a->key_heads);
        p.n_ctx = (int32_t)a->t, p.n_keys = (int32_t)a->n, p.k_lengths = a->lengths;
        p.splits = plan.splits;
        p.q_blocks = (int32_t)((a->t + plan.e->bm - 1) / plan.e->bm);
        const int64_t nmb = (int64_t)p.q_blocks * p.group * p.splits;
        if (nmb * p.num_heads > (int64_t(1) << 30)) return RSFA_E_CROSS;
        p.nmb = (int32_t)nmb;
        p.num_tasks = p.num_heads * p.nmb;
        p.c = c, p.neg = a->sm_scale < 0.0f ? 1u : 0u;
        p.part_o = part_o, p.part_ml = part_ml;
        if (plan.splits > 1) p.lse = nullptr;
        if ((st = launch_cross(*plan.e, p, stream)) != RSFA_OK) return st;
    }
    if (plan.splits == 1) return RSFA_OK;
    JoinParams j{};
    j.part_o = part_o, j.part_ml = part_ml, j.o = a->o, j.lse = a->lse, j.lengths = a->lengths;
    for (int i = 0; i < 3; ++i) j.o_st[i] = a->o_stride[i];
    j.heads = (int32_t)a->heads, j.t = (int32_t)a->t, j.splits = plan.splits;
    j.rows = a->z * a->heads * a->t;
    const int groups = 256 / (int)(a->head_dim / 4);
    j.pp = 1;
    while (j.pp < groups && j.pp * 8 < plan.splits) j.pp *= 2;
    const int64_t per = groups / j.pp, blocks = (j.rows + per - 1) / per;
    if (blocks > 0x7fffffff) return RSFA_E_CROSS;
    void* args[] = {&j};
    return hipLaunchKernel(bf16 ? join_fn<TypeBF16>(a->head_dim) : join_fn<TypeF16>(a->head_dim), dim3((unsigned)blocks), dim3(256), args, 0,
                           (hipStream_t)stream) == hipSuccess ? RSFA_OK : RSFA_E_LAUNCH;
}

}  // extern "C"
