// Attention over a 4-bit cache (rsfa_cache4_attend, declared in include/rsfa.h).
//
//   s = sm_scale q k^T,  o = softmax(s) v,  weight[slot] += sum over rows of softmax(s)[slot]
//
// The rows that share a key head (the query heads of its group, all tokens) are
// row = token * group + head, and a wave holds NB blocks of 16 of them.  Codes
// go from global memory into registers, are converted to the cache's type by
// v_cvt_scalef32_pk_{f16,bf16}_fp4 (exact: two significant bits and a power of
// two) and into v_mfma_f32_16x16x32; neither K, V nor the softmax weights pass through LDS:
//   S^T = K Q^T  A: lane l has the key l % 16 and the D/4 consecutive values that
//                start at (l / 16) * D/4, so a key tile of 16 is one load of D/8
//                bytes a lane (D = 128: one 16-byte load, one block, one scale).
//                B: the row l % 16 of Q, the same values.
//   O^T = V^T P^T  in S^T's accumulator, lane l holds the row l % 16 and the keys
//                4 * (l / 16) + r of each 16-key tile; as the k index of B only
//                has to agree with A's, the P values go into B where they
//                are: k = 8 * (l / 16) + 4 * t + r is key 16 * t + 4 * (l / 16) + r.
//                A: lane l has these 8 keys of the D/16 consecutive values that
//                start at (l % 16) * D/16: a load of D/32 bytes per key, converted in
//                pairs of values and paired by key with v_perm_b32.
// Statistics, sums and accumulators are in 32 bits.  The running maximum of a row
// only moves when a score passes it by SLACK (log2 units), as the weights then
// stay below 2^SLACK and the final division takes the factor out; the row
// sum adds the weights before they are rounded to the cache's type for P V.
#include "cache4.hpp"

using namespace rsfa4;

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float SLACK = 8.0f;
// Start of a row's running maximum: below every finite score, and finite, so
// that a hidden score's exp2(-inf - m) is 0 and not NaN.
constexpr float NEVER = -3.0e38f;
constexpr int TILE = 32;  // keys of a wave's step

struct AttendParams {
    rsfa_cache4 c;
    const char* q;
    char* o;
    float* lse;
    int64_t qs[3], os[3];      // element strides of (Z, heads, T)
    int32_t heads, group, t;   // query heads, query heads per key head, tokens
    int32_t rows;              // group * t
    const int32_t *lengths, *counts, *pos_start;
    int64_t length;
    int32_t most;              // slots that may be read
    int32_t bh;                // Z * H
    int32_t splits;            // parts that a sequence's slots are split into
    float scale;               // |sm_scale| * log2 e
    uint32_t neg;              // sign of sm_scale, as a mask for a pair of q's values
    float* part_o;             // [splits][bh][rows][D] (splits > 1)
    float2* part_ml;           // [splits][bh][rows]: maximum (log2 units), sum
    float* scores;             // [bh][rows][most]: scores in log2 units, or null
    float* row_lse;            // [bh][rows]: log2 of the row's sum of exp2 (weights of many rows)
};

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, typename T::x2));
}

// Byte I of the scale bytes in `w`, as a float whose exponent it is (the other
// bits are whatever lies beside it).
__device__ __forceinline__ float scale_bits(uint32_t w, int byte) {
    return __uint_as_float(__builtin_amdgcn_alignbit(w, w, (8 * byte + 9) & 31));
}

template <int BYTES>
struct Bytes;
template <> struct Bytes<1> { typedef uint8_t type; };
template <> struct Bytes<2> { typedef uint16_t type; };
template <> struct Bytes<4> { typedef uint32_t type; };

// A wave's raw K and V tile of 32 keys.
template <int D>
struct Raw {
    static constexpr int KW = D / 32;             // dwords of K codes a lane has of a key
    static constexpr int VW = D >= 128 ? D / 128 : 1;  // dwords of V codes a lane has of a key
    uint32_t k[2][KW];
    uint32_t ks[2];                               // scale bytes of the lane's K values (byte 0, 1 at D = 256)
    uint32_t v[8][VW];
    uint32_t vs[8];                               // D >= 128: the dword of the key's scale bytes that has the lane's
};

template <int D>
struct Loader {
    const uint8_t *kc, *ks, *vc, *vs;  // of the sequence and head
    int lane, col, grp;

    // Slots past `last` read slot `last` (TAIL) or are known to exist.
    template <bool TAIL>
    __device__ __forceinline__ void load(Raw<D>& r, int tile, int last) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int key = tile + 16 * h + col;
            if (TAIL) key = min(key, last);
            const uint8_t* p = kc + (int64_t)key * (D / 2) + grp * (D / 8);
            if constexpr (D == 32) {
                r.k[h][0] = *(const uint32_t*)p;
            } else if constexpr (D == 64) {
                const u32x2 w = *(const u32x2*)p;
                r.k[h][0] = w[0], r.k[h][1] = w[1];
            } else {
#pragma unroll
                for (int i = 0; i < D / 128; ++i) {
                    const u32x4 w = *(const u32x4*)(p + 16 * i);
#pragma unroll
                    for (int j = 0; j < 4; ++j) r.k[h][4 * i + j] = w[j];
                }
            }
            const uint8_t* s = ks + (int64_t)key * (D / 32);
            if constexpr (D == 256) r.ks[h] = *(const uint16_t*)(s + 2 * grp);
            else r.ks[h] = s[grp * (D / 4) / 32];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            int key = tile + 16 * (j / 4) + 4 * grp + j % 4;
            if (TAIL) key = min(key, last);
            const uint8_t* p = vc + (int64_t)key * (D / 2) + col * (D / 32);
            if constexpr (D == 256) {
                const u32x2 w = *(const u32x2*)p;
                r.v[j][0] = w[0], r.v[j][1] = w[1];
            } else {
                r.v[j][0] = *(const typename Bytes<D / 32>::type*)p;
            }
            const uint8_t* s = vs + (int64_t)key * (D / 32);
            if constexpr (D == 256) r.vs[j] = *(const uint32_t*)(s + (col / 8) * 4);
            else r.vs[j] = *(const typename Bytes<D / 32>::type*)s;
        }
    }
    // The byte of vs[] that scales the lane's V values.
    __device__ __forceinline__ int v_byte() const {
        return D == 256 ? (col / 2) & 3 : D == 128 ? col / 4 : D == 64 ? col / 8 : 0;
    }
};

// NB blocks of 16 rows a wave; RW of the workgroup's four waves take rows of
// their own, the others share their rows' keys.
template <class T, int D, int NB, int RW>
struct Geometry {
    static constexpr int KWAVES = 4 / RW;
    static constexpr int ROWS = RW * NB * 16;
};

template <class T, int D, int NB, int RW, bool CAUSAL>
__global__ void __launch_bounds__(256, 2) attend_kernel(AttendParams p) {
    typedef Geometry<T, D, NB, RW> G;
    typedef typename T::x8 x8;
    typedef typename T::elem elem;
    constexpr int DT = D / 16;  // 16-row tiles of O^T
    constexpr int QS = D / 32;  // k steps of S^T
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, grp = lane >> 4;
    const int rw = wave / G::KWAVES, kw = wave % G::KWAVES;
    const int bh = blockIdx.x % p.bh;  // with a multiple of 8, a head's row tiles meet in one XCD's L2
    const int tile_id = blockIdx.x / p.bh;
    const int split = blockIdx.y;
    const int z = bh / (int)p.c.h, h = bh - z * (int)p.c.h;
    const int len = length_of(p.lengths, p.length, z, p.most);
    const int count = p.counts ? max(0, min(p.counts[z], p.t)) : p.t;
    const int row0 = tile_id * G::ROWS + rw * NB * 16;

    Loader<D> ld;
    {
        const int64_t c = z * p.c.code_stride[0] + h * p.c.code_stride[1];
        const int64_t s = z * p.c.scale_stride[0] + h * p.c.scale_stride[1];
        ld.kc = p.c.k_codes + c, ld.vc = p.c.v_codes + c;
        ld.ks = p.c.k_scales + s, ld.vs = p.c.v_scales + s;
        ld.lane = lane, ld.col = col, ld.grp = grp;
    }
    const int32_t* pos = p.c.positions + z * p.c.slot_stride[0] + h * p.c.slot_stride[1];

    // Q^T and the rows' positions
    x8 q[NB][QS];
    int qpos[NB];
    int least = 0x7fffffff, greatest = -0x7fffffff - 1;  // of the wave's valid rows' positions
    bool any_row = false;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int row = row0 + 16 * b + col;
        const int tok = row / p.group, head = row - tok * p.group;
        const bool valid = tok < count;  // (row < rows follows)
        any_row |= valid;
        u32x4 w[QS] = {};
        if (valid) {
            const elem* src = (const elem*)p.q + z * p.qs[0] + (int64_t)(h * p.group + head) * p.qs[1] + tok * p.qs[2] + grp * (D / 4);
#pragma unroll
            for (int i = 0; i < QS; ++i) w[i] = *(const u32x4*)(src + 8 * i);
        }
#pragma unroll
        for (int i = 0; i < QS; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[i][j] ^= p.neg;
            q[b][i] = __builtin_bit_cast(x8, w[i]);
        }
        if (CAUSAL) {
            const int64_t at = (p.pos_start ? (int64_t)p.pos_start[z] : (int64_t)len - count) + tok;
            qpos[b] = (int)(at > 0x7fffffff ? 0x7fffffff : at);
            if (valid) least = min(least, qpos[b]), greatest = max(greatest, qpos[b]);
        }
    }
    if (CAUSAL) {
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
            least = min(least, __shfl_xor(least, d));
            greatest = max(greatest, __shfl_xor(greatest, d));
        }
    }

    f32x4 acc[NB][DT];
    float m[NB], l[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        m[b] = NEVER;
        l[b] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[b][d] = (f32x4){0, 0, 0, 0};
    }

    // this split's keys, a whole number of tiles for every wave but the last's
    const int step = TILE * G::KWAVES;
    const int chunk = ((len + p.splits - 1) / p.splits + step - 1) / step * step;
    const int64_t start64 = (int64_t)chunk * split;
    const int start = (int)(start64 < len ? start64 : len);
    const int end = min(start + chunk, len);
    const int vbyte = ld.v_byte();

    auto compute = [&](const Raw<D>& r, int tile) {
        // hidden keys: past the end, or (causal) of a later position than a row's
        int kpos[8];
        bool masked = tile + TILE > end;
        if (CAUSAL) {
            int far = -0x7fffffff - 1, near = 0x7fffffff;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = tile + 16 * (j / 4) + 4 * grp + j % 4;
                kpos[j] = pos[min(key, len - 1)];
                far = max(far, kpos[j]);
                near = min(near, kpos[j]);
            }
            masked |= __any(far > least);
            if (!__any(near <= greatest)) {
                if (p.scores) {  // no row sees the tile: its scores all the same are read
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const int row = row0 + 16 * b + col;
                        if (row < p.rows)
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const int key = tile + 16 * (j / 4) + 4 * grp + j % 4;
                                if (key < end) p.scores[((int64_t)bh * p.rows + row) * p.most + key] = -INFINITY;
                            }
                    }
                }
                return;
            }
        }
        f32x4 s[NB][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const float sc0 = scale_bits(r.ks[t], 0), sc1 = scale_bits(r.ks[t], 1);
#pragma unroll
            for (int b = 0; b < NB; ++b) s[b][t] = (f32x4){0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < QS; ++i) {
                const uint32_t w = r.k[t][i];
                const float sc = D == 256 && i >= 4 ? sc1 : sc0;
                const u32x4 kv = {T::template cvt<0>(w, sc), T::template cvt<1>(w, sc), T::template cvt<2>(w, sc),
                                  T::template cvt<3>(w, sc)};
#pragma unroll
                for (int b = 0; b < NB; ++b) s[b][t] = T::mfma(__builtin_bit_cast(x8, kv), q[b][i], s[b][t]);
            }
        }
        uint32_t pk[NB][4];
        uint32_t visible[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float x[8];
            visible[b] = 0xff;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = s[b][j / 4][j % 4] * p.scale;
            if (masked) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int key = tile + 16 * (j / 4) + 4 * grp + j % 4;
                    const bool hidden = key >= end || (CAUSAL && kpos[j] > qpos[b]);
                    if (hidden) x[j] = -INFINITY, visible[b] &= ~(1u << j);
                }
            }
            if (p.scores) {
                const int row = row0 + 16 * b + col;
                if (row < p.rows) {
                    float* dst = p.scores + ((int64_t)bh * p.rows + row) * p.most + tile + 4 * grp;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (!masked || tile + 16 * (j / 4) + 4 * grp + j % 4 < end) dst[16 * (j / 4) + j % 4] = x[j];
                }
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
            for (int j = 0; j < 4; ++j) pk[b][j] = pack2<T>(x[2 * j], x[2 * j + 1]);
        }
        // V's scales; where a row of the tile does not see every key, a NaN block
        // must not reach it (0 * NaN): it is scaled as 0 and put into the rows that see it
        float sc[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) sc[j] = scale_bits(r.vs[j], vbyte);
        if (masked) {
            uint32_t bad = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if ((__float_as_uint(sc[j]) & 0x7f800000u) == 0x7f800000u) bad |= 1u << j, sc[j] = 0.0f;
            if (__any(bad != 0)) {
                // lane l's O^T values are rows 4 (l / 16) + r of each tile: dims
                // (4 (l / 16) + r) D/16 + d, whose block is that of a lane with col = 4 (l / 16) + r
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        bool hit = false;
                        for (int g = 0; g < 4; ++g) {
                            const uint32_t vis = __shfl((int)visible[b], 16 * g + col);
                            const uint32_t there = __shfl((int)bad, 16 * g + 4 * grp + i);
                            hit |= (vis & there) != 0;
                        }
                        if (hit)
#pragma unroll
                            for (int d = 0; d < DT; ++d) acc[b][d][i] = __builtin_nanf("");
                    }
            }
        }
#pragma unroll
        for (int pr = 0; pr < D / 32; ++pr) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t c = r.v[j][pr / 4];
                w[j] = pr % 4 == 0   ? T::template cvt<0>(c, sc[j])
                       : pr % 4 == 1 ? T::template cvt<1>(c, sc[j])
                       : pr % 4 == 2 ? T::template cvt<2>(c, sc[j])
                                     : T::template cvt<3>(c, sc[j]);
            }
            u32x4 even, odd;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                even[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x05040100u);
                odd[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x07060302u);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const x8 pb = __builtin_bit_cast(x8, (u32x4){pk[b][0], pk[b][1], pk[b][2], pk[b][3]});
                acc[b][2 * pr] = T::mfma(__builtin_bit_cast(x8, even), pb, acc[b][2 * pr]);
                acc[b][2 * pr + 1] = T::mfma(__builtin_bit_cast(x8, odd), pb, acc[b][2 * pr + 1]);
            }
        }
    };

    // (a wave whose rows are all invalid still takes part in the exchange below)
    if (__any(any_row)) {
        int tile = start + TILE * kw;
        if (tile < end) {
            Raw<D> cur, next;
            if (tile + TILE <= len) ld.template load<false>(cur, tile, 0);
            else ld.template load<true>(cur, tile, len - 1);
            for (;;) {
                const int after = tile + step;
                if (after < end) {
                    if (after + TILE <= len) ld.template load<false>(next, after, 0);
                    else ld.template load<true>(next, after, len - 1);
                }
                compute(cur, tile);
                if (after >= end) break;
                cur = next;
                tile = after;
            }
        }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        l[b] += __shfl_xor(l[b], 16);
        l[b] += __shfl_xor(l[b], 32);
        // rows past the count are empty (their q was taken as 0)
        if ((row0 + 16 * b + col) / p.group >= count) m[b] = NEVER, l[b] = 0.0f;
    }

    if constexpr (G::KWAVES > 1) {
        // the waves that share rows add up their parts, through LDS
        constexpr int PITCH = D + 4;  // dwords of a row: 16-lane columns meet no bank twice
        __shared__ float2 ml[4][NB * 16];
        __shared__ float part[RW][NB * 16][PITCH];
#pragma unroll
        for (int b = 0; b < NB; ++b)
            if (grp == 0) ml[wave][16 * b + col] = make_float2(m[b], l[b]);
        __syncthreads();
        float f[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float mm = NEVER, ll = 0.0f;
            for (int k = 0; k < G::KWAVES; ++k) mm = fmaxf(mm, ml[rw * G::KWAVES + k][16 * b + col].x);
            for (int k = 0; k < G::KWAVES; ++k) {
                const float2 v = ml[rw * G::KWAVES + k][16 * b + col];
                ll += v.y * __builtin_amdgcn_exp2f(v.x - mm);
            }
            f[b] = __builtin_amdgcn_exp2f(m[b] - mm);
            m[b] = mm;
            l[b] = ll;
        }
        for (int k = G::KWAVES - 1; k >= 0; --k) {
            if (kw == k) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float* at = &part[rw][16 * b + col][(4 * grp + i) * DT];
#pragma unroll
                        for (int d = 0; d < DT; ++d) {
                            float v = acc[b][d][i] * f[b];
                            if (k < G::KWAVES - 1) v += at[d];
                            if (k > 0) at[d] = v;
                            else acc[b][d][i] = v;
                        }
                    }
            }
            __syncthreads();
        }
        if (kw != 0) return;
    }

#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int row = row0 + 16 * b + col;
        if (row >= p.rows) continue;
        const int tok = row / p.group, head = row - tok * p.group;
        if (p.splits > 1) {
            const int64_t at = ((int64_t)split * p.bh + bh) * p.rows + row;
            if (grp == 0) p.part_ml[at] = make_float2(m[b], l[b]);
            float* dst = p.part_o + at * D;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int d = 0; d < DT; d += 2)
                    *(float2*)(dst + (4 * grp + i) * DT + d) = make_float2(acc[b][d][i], acc[b][d + 1][i]);
            continue;
        }
        // (a NaN sum is a row whose scores are NaN)
        const float inv = l[b] == 0.0f ? 0.0f : 1.0f / l[b];
        const int64_t hq = h * p.group + head;
        elem* dst = (elem*)p.o + z * p.os[0] + hq * p.os[1] + tok * p.os[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w[DT / 2];
#pragma unroll
            for (int d = 0; d < DT; d += 2)
                w[d / 2] = l[b] == 0.0f ? 0u : pack2<T>(acc[b][d][i] * inv, acc[b][d + 1][i] * inv);
            elem* at = dst + (4 * grp + i) * DT;
#pragma unroll
            for (int d = 0; d < DT / 2; ++d) ((uint32_t*)at)[d] = w[d];
        }
        if (grp == 0) {
            const float lse2 = l[b] == 0.0f ? -INFINITY : m[b] + __builtin_amdgcn_logf(l[b]);
            if (p.lse) p.lse[(z * (int64_t)p.heads + hq) * p.t + tok] = lse2 * LN2;
            if (p.row_lse) p.row_lse[(int64_t)bh * p.rows + row] = lse2;
        }
    }
}

// Sum of a row's parts: one wave a row.
template <class T, int D>
__global__ void __launch_bounds__(256) join_kernel(AttendParams p) {
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);  // bh * rows + row
    const int lane = threadIdx.x & 63;
    const int64_t all = (int64_t)p.bh * p.rows;
    if (id >= all) return;
    const int bh = (int)(id / p.rows), row = (int)(id - (int64_t)bh * p.rows);
    float m = NEVER;
    for (int s = lane; s < p.splits; s += 64) m = fmaxf(m, p.part_ml[s * all + id].x);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    constexpr int W = D >= 64 ? D / 64 : 1;
    float o[W] = {};
    float l = 0.0f;
    const bool mine = lane * W < D;
    for (int s = 0; s < p.splits; ++s) {
        const float2 v = p.part_ml[s * all + id];
        if (v.y == 0.0f) continue;  // no slot in this part
        const float f = __builtin_amdgcn_exp2f(v.x - m);
        l += v.y * f;
        if (mine)
#pragma unroll
            for (int i = 0; i < W; ++i) o[i] += p.part_o[(s * all + id) * D + lane * W + i] * f;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int z = bh / (int)p.c.h, h = bh - z * (int)p.c.h;
    const int tok = row / p.group, head = row - tok * p.group;
    const int64_t hq = h * p.group + head;
    typename T::elem* dst = (typename T::elem*)p.o + z * p.os[0] + hq * p.os[1] + tok * p.os[2] + lane * W;
    if (mine)
#pragma unroll
        for (int i = 0; i < W; ++i) dst[i] = (typename T::elem)(o[i] * inv);
    if (lane == 0) {
        const float lse2 = l == 0.0f ? -INFINITY : m + __builtin_amdgcn_logf(l);
        if (p.lse) p.lse[(z * (int64_t)p.heads + hq) * p.t + tok] = lse2 * LN2;
        if (p.row_lse) p.row_lse[id] = lse2;
    }
}

// Weights of few rows: from their scores and sums.  A thread takes four slots.
__global__ void __launch_bounds__(256) add_weights_kernel(AttendParams p) {
    const int bh = blockIdx.x % p.bh;
    const int z = bh / (int)p.c.h, h = bh - z * (int)p.c.h;
    const int len = length_of(p.lengths, p.length, z, p.most);
    const int count = p.counts ? max(0, min(p.counts[z], p.t)) : p.t;
    const int rows = count * p.group;
    float* w = p.c.weights + z * p.c.slot_stride[0] + h * p.c.slot_stride[1];
    for (int i = 0; i < 4; ++i) {
        const int64_t slot = (int64_t)(blockIdx.x / p.bh) * 1024 + 256 * i + threadIdx.x;
        if (slot >= len) return;
        float sum = 0.0f;
        for (int r = 0; r < rows; ++r) {
            const float lse2 = p.row_lse[(int64_t)bh * p.rows + r];
            // (a row that sees no slot has -inf)
            if (lse2 != -INFINITY) sum += __builtin_amdgcn_exp2f(p.scores[((int64_t)bh * p.rows + r) * p.most + slot] - lse2);
        }
        w[slot] += sum;
    }
}

// Weights of many rows: the scores are computed again, now that the rows' sums
// are known.  A workgroup holds 64 keys in registers, each wave all of them,
// and its waves take every fourth block of 16 rows.
template <class T, int D, bool CAUSAL>
__global__ void __launch_bounds__(256, 2) weights_kernel(AttendParams p) {
    constexpr int KT = 4;  // tiles of 16 keys
    constexpr int QS = D / 32;
    typedef typename T::x8 x8;
    typedef typename T::elem elem;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, grp = lane >> 4;
    const int bh = blockIdx.x % p.bh;
    const int z = bh / (int)p.c.h, h = bh - z * (int)p.c.h;
    const int len = length_of(p.lengths, p.length, z, p.most);
    const int count = p.counts ? max(0, min(p.counts[z], p.t)) : p.t;
    const int64_t tile = (int64_t)(blockIdx.x / p.bh) * (16 * KT);
    if (tile >= len) return;
    const uint8_t* kc = p.c.k_codes + z * p.c.code_stride[0] + h * p.c.code_stride[1];
    const uint8_t* ks = p.c.k_scales + z * p.c.scale_stride[0] + h * p.c.scale_stride[1];
    const int32_t* pos = p.c.positions + z * p.c.slot_stride[0] + h * p.c.slot_stride[1];
    x8 k[KT][QS];
    int kpos[CAUSAL ? KT : 1][4];
    int far = -0x7fffffff - 1, near = 0x7fffffff;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        const int key = (int)min(tile + 16 * t + col, (int64_t)len - 1);
        const uint8_t* s = ks + (int64_t)key * (D / 32);
        uint32_t sw;
        if constexpr (D == 256) sw = *(const uint16_t*)(s + 2 * grp);
        else sw = s[grp * (D / 4) / 32];
        const float sc0 = scale_bits(sw, 0), sc1 = scale_bits(sw, 1);
#pragma unroll
        for (int i = 0; i < QS; ++i) {
            const uint32_t w = *(const uint32_t*)(kc + (int64_t)key * (D / 2) + grp * (D / 8) + 4 * i);
            const float sc = D == 256 && i >= 4 ? sc1 : sc0;
            const u32x4 kv = {T::template cvt<0>(w, sc), T::template cvt<1>(w, sc), T::template cvt<2>(w, sc),
                              T::template cvt<3>(w, sc)};
            k[t][i] = __builtin_bit_cast(x8, kv);
        }
        if (CAUSAL)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int v = pos[min(tile + 16 * t + 4 * grp + r, (int64_t)len - 1)];
                kpos[t][r] = v;
                far = max(far, v);
                near = min(near, v);
            }
    }
    if (CAUSAL) {
#pragma unroll
        for (int d = 16; d < 64; d <<= 1) {
            far = max(far, __shfl_xor(far, d));
            near = min(near, __shfl_xor(near, d));
        }
    }
    float sum[KT][4] = {};
    const int64_t first = CAUSAL ? (p.pos_start ? (int64_t)p.pos_start[z] : (int64_t)len - count) : 0;
    const int rows = count * p.group;
    for (int row0 = 16 * wave; row0 < rows; row0 += 64) {
        const int row = row0 + col;
        const int tok = min(row, rows - 1) / p.group, head = min(row, rows - 1) - tok * p.group;
        int qpos = 0;
        bool masked = row0 + 16 > rows;
        if (CAUSAL) {
            const int64_t at = first + tok;
            qpos = (int)(at > 0x7fffffff ? 0x7fffffff : at);
            // the block's rows have positions that grow with the row
            const int64_t lo = first + row0 / p.group, hi = first + (min(row0 + 16, rows) - 1) / p.group;
            if (near > hi) continue;
            masked |= far > lo;
        }
        const float lse2 = row < rows ? p.row_lse[(int64_t)bh * p.rows + row] : -INFINITY;
        masked |= __any(lse2 == -INFINITY);
        const elem* src = (const elem*)p.q + z * p.qs[0] + (int64_t)(h * p.group + head) * p.qs[1] + tok * p.qs[2] + grp * (D / 4);
        x8 q[QS];
#pragma unroll
        for (int i = 0; i < QS; ++i) {
            u32x4 w = *(const u32x4*)(src + 8 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] ^= p.neg;
            q[i] = __builtin_bit_cast(x8, w);
        }
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            f32x4 s = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < QS; ++i) s = T::mfma(k[t][i], q[i], s);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float x = __builtin_amdgcn_exp2f(s[r] * p.scale - lse2);
                if (masked) x = lse2 == -INFINITY || (CAUSAL && kpos[t][r] > qpos) ? 0.0f : x;
                sum[t][r] += x;
            }
        }
    }
    __shared__ float total[4][16 * KT];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float v = sum[t][r];
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) v += __shfl_xor(v, d);
            if (col == 0) total[wave][16 * t + 4 * grp + r] = v;
        }
    __syncthreads();
    const int i = threadIdx.x;
    if (i < 16 * KT && tile + i < len) {
        float* w = p.c.weights + z * p.c.slot_stride[0] + h * p.c.slot_stride[1];
        w[tile + i] += (total[0][i] + total[1][i]) + (total[2][i] + total[3][i]);
    }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
struct Plan {
    int nb, rw;        // blocks of 16 rows a wave, waves with rows of their own
    int tiles, splits;
    bool scores;       // weights from stored scores
    uint64_t part_o, part_ml, scores_at, row_lse, bytes;  // offsets into the workspace
};

// Rows up to 32 share their keys among the four waves of a workgroup; more give
// each wave 32 rows of its own.
Plan make_plan(const rsfa_cache4_attend_args* a, int cus) {
    Plan p{};
    const int64_t group = a->heads / a->cache.h, rows = group * a->t;
    const int64_t bh = a->cache.z * a->cache.h;
    const int64_t most = a->max_length > 0 && a->max_length < a->cache.capacity ? a->max_length : a->cache.capacity;
    const bool few = rows <= 16 || (rows <= 32 && a->cache.head_dim <= 128);
    p.nb = rows <= 16 || (!few && a->cache.head_dim == 256) ? 1 : 2;
    p.rw = few ? 1 : 4;
    const int per = p.rw * p.nb * 16;
    p.tiles = (int)((rows + per - 1) / per);
    // enough workgroups for the chip, of at least four steps each
    const int64_t step = TILE * (4 / p.rw);
    const int64_t want = (4 * (int64_t)cus + bh * p.tiles - 1) / (bh * p.tiles);
    const int64_t able = (most + 4 * step - 1) / (4 * step);
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, able), 256));
    p.scores = a->accumulate && few;
    uint64_t at = 0;
    auto take = [&](uint64_t n) {
        const uint64_t here = at;
        at += (n + 255) / 256 * 256;
        return here;
    };
    if (p.splits > 1) {
        p.part_o = take((uint64_t)p.splits * bh * rows * a->cache.head_dim * 4);
        p.part_ml = take((uint64_t)p.splits * bh * rows * 8);
    }
    if (a->accumulate) p.row_lse = take((uint64_t)bh * rows * 4);
    if (p.scores) p.scores_at = take((uint64_t)bh * rows * most * 4);
    p.bytes = at;
    return p;
}

int cus_of_current_device() {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1)
        return 256;
    return n;
}

template <class T, int D, bool CAUSAL>
const void* attend_fn(const Plan& p) {
    if (p.rw == 1) {
        if constexpr (D <= 128)
            if (p.nb == 2) return (const void*)&attend_kernel<T, D, 2, 1, CAUSAL>;
        return (const void*)&attend_kernel<T, D, 1, 1, CAUSAL>;
    }
    if constexpr (D <= 128) return (const void*)&attend_kernel<T, D, 2, 4, CAUSAL>;
    else return (const void*)&attend_kernel<T, D, 1, 4, CAUSAL>;
}

struct Functions {
    const void *attend, *join, *weights;
};

template <class T, int D>
Functions functions(const Plan& p, bool causal) {
    return {causal ? attend_fn<T, D, true>(p) : attend_fn<T, D, false>(p), (const void*)&join_kernel<T, D>,
            causal ? (const void*)&weights_kernel<T, D, true> : (const void*)&weights_kernel<T, D, false>};
}

template <class T>
Functions functions(const Plan& p, bool causal, int64_t d) {
    switch (d) {
        case 32: return functions<T, 32>(p, causal);
        case 64: return functions<T, 64>(p, causal);
        case 128: return functions<T, 128>(p, causal);
        default: return functions<T, 256>(p, causal);
    }
}

int check_attend(const rsfa_cache4_attend_args* a) {
    if (!a) return RSFA_E_NULL;
    if (a->struct_size != sizeof(rsfa_cache4_attend_args)) return RSFA_E_ABI;
    int st = check_cache(a->cache, a->accumulate != 0);
    if (st != RSFA_OK) return st;
    if (a->heads < 1 || a->heads % a->cache.h || a->heads > (1 << 24) || a->t < 1 || a->t > (1 << 24) ||
        a->heads / a->cache.h * a->t > (1 << 28) || a->max_length < 0)
        return RSFA_E_CACHE;
    return RSFA_OK;
}

}  // namespace

extern "C" {

uint64_t rsfa_cache4_attend_workspace_bytes(const rsfa_cache4_attend_args* a) {
    if (check_attend(a) != RSFA_OK) return 0;
    return make_plan(a, cus_of_current_device()).bytes;
}

int rsfa_cache4_attend(const rsfa_cache4_attend_args* a, void* stream) {
    int st = check_attend(a);
    if (st != RSFA_OK) return st;
    if (!a->q || !a->o) return RSFA_E_NULL;
    if ((st = check_rows(a->q, a->q_stride)) != RSFA_OK || (st = check_rows(a->o, a->o_stride)) != RSFA_OK) return st;
    if (((uintptr_t)a->lse | (uintptr_t)a->lengths | (uintptr_t)a->counts | (uintptr_t)a->pos_start) & 3)
        return RSFA_E_ALIGN;
    const Plan plan = make_plan(a, cus_of_current_device());
    if (plan.bytes) {
        if (!a->workspace || a->workspace_bytes < plan.bytes) return RSFA_E_WORKSPACE;
        if ((uintptr_t)a->workspace & 15) return RSFA_E_ALIGN;
    }
    AttendParams p{};
    p.c = a->cache;
    p.q = (const char*)a->q, p.o = (char*)a->o, p.lse = a->lse;
    for (int i = 0; i < 3; ++i) p.qs[i] = a->q_stride[i], p.os[i] = a->o_stride[i];
    p.heads = (int32_t)a->heads;
    p.group = (int32_t)(a->heads / a->cache.h);
    p.t = (int32_t)a->t;
    p.rows = p.group * p.t;
    p.lengths = a->lengths, p.counts = a->counts, p.pos_start = a->pos_start;
    p.length = a->length;
    p.most = (int32_t)(a->max_length > 0 && a->max_length < a->cache.capacity ? a->max_length : a->cache.capacity);
    p.bh = (int32_t)(a->cache.z * a->cache.h);
    p.splits = plan.splits;
    p.scale = __builtin_fabsf(a->sm_scale) * LOG2E;
    p.neg = a->sm_scale < 0.0f ? 0x80008000u : 0u;
    char* ws = (char*)a->workspace;
    if (plan.splits > 1) {
        p.part_o = (float*)(ws + plan.part_o);
        p.part_ml = (float2*)(ws + plan.part_ml);
    }
    if (a->accumulate) p.row_lse = (float*)(ws + plan.row_lse);
    if (plan.scores) p.scores = (float*)(ws + plan.scores_at);
    const bool causal = a->causal != 0;
    const Functions fn = a->cache.dtype == RSFA_DTYPE_BF16 ? functions<BF16>(plan, causal, a->cache.head_dim)
                                                           : functions<F16>(plan, causal, a->cache.head_dim);
    const int64_t grid = (int64_t)p.bh * plan.tiles;
    const int64_t slots = plan.scores ? 1024 : 64;
    const int64_t weight_grid = (int64_t)p.bh * ((p.most + slots - 1) / slots);
    if (grid > 0x7fffffff || (a->accumulate && weight_grid > 0x7fffffff)) return RSFA_E_CACHE;
    void* args[] = {&p};
    if (hipLaunchKernel(fn.attend, dim3((unsigned)grid, (unsigned)plan.splits), dim3(256), args, 0, (hipStream_t)stream) != hipSuccess)
        return RSFA_E_LAUNCH;
    if (plan.splits > 1) {
        const int64_t rows = (int64_t)p.bh * p.rows;
        if (hipLaunchKernel(fn.join, dim3((unsigned)((rows + 3) / 4)), dim3(256), args, 0, (hipStream_t)stream) != hipSuccess)
            return RSFA_E_LAUNCH;
    }
    if (a->accumulate) {
        const void* f = plan.scores ? (const void*)&add_weights_kernel : fn.weights;
        if (hipLaunchKernel(f, dim3((unsigned)weight_grid), dim3(256), args, 0, (hipStream_t)stream) != hipSuccess)
            return RSFA_E_LAUNCH;
    }
    return RSFA_OK;
}

}  // extern "C"
