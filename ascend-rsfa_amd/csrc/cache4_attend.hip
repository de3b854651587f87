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
// stay below 2^SLACK and the final division takes the factor out.  A weight is rounded to the
// cache's type for P V, half a step at most, as the matrix unit takes 16-bit operands at sixteen times
// the rate of 32-bit ones; the row sum, lse and the slots' weights take it unrounded.  (o is then about 1.35
// times as far from 64 bits as with 32-bit weights, most of either distance being o's own rounding.)
#include <cfloat>
#include <type_traits>

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
constexpr int NAN_OR_INF = 0x207;  // class mask: an exponent of all ones, as a scale byte of 255 gives

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
    float* row_lse;            // [bh][rows]: log2 of the row's sum of exp2 (for the weights)
    float* part_w;             // [parts][bh][most]: sums of parts of the rows, or null
    const uint32_t* tree;      // MASK_TREE: [Z][t][tree_words]: the drafted tokens that a token sees
    int64_t tree_sz;           // its stride of Z (0: one tree for all)
    int32_t tree_words;
};

// What a row sees of the slots in use: all of them; those of a position up to its own; or those before the
// call's drafted tokens, which are the last `count` slots in use, and of these the ones whose bit its token has.
enum { MASK_NONE = 0, MASK_POSITION = 1, MASK_TREE = 2 };

// The 32 slots whose first is the drafted token `first` (below 0: slots of the context, all seen), as a mask,
// from the bits of a token.  A token past the bits' last word is seen by none.
__device__ __forceinline__ uint32_t tree_mask(const uint32_t* bits, int words, int first) {
    const int w = first >> 5;  // (rounds down)
    const uint32_t lo = w < 0 ? 0xffffffffu : w < words ? bits[w] : 0u;
    const uint32_t hi = w + 1 < 0 ? 0xffffffffu : w + 1 < words ? bits[w + 1] : 0u;
    return __builtin_amdgcn_alignbit(hi, lo, first & 31);
}

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

typedef u32x4 u32x4_u __attribute__((aligned(4)));  // loads need the alignment of a dword
typedef f32x4 f32x4_u __attribute__((aligned(4)));
// scale rows of two bytes and of one
typedef u32x2 u32x2_u __attribute__((aligned(2)));
typedef uint32_t u32_u __attribute__((aligned(1)));

template <int BYTES>
struct Bytes;
template <> struct Bytes<1> { typedef uint8_t type; };
template <> struct Bytes<2> { typedef uint16_t type; };
template <> struct Bytes<4> { typedef uint32_t type; };

// A wave's raw K and V tile of 32 keys.
template <int D, bool CAUSAL>
struct Raw {
    static constexpr int KW = D / 32;             // dwords of K codes a lane has of a key
    static constexpr int VW = D >= 128 ? D / 128 : 1;  // dwords of V codes a lane has of a key
    uint32_t k[2][KW];
    uint32_t ks[2];                               // scale bytes of the lane's K values (byte 0, 1 at D = 256)
    uint32_t v[8][VW];
    static constexpr int SW = D >= 128 ? 1 : 128 / D;  // V keys whose scale bytes share a dword
    uint32_t vs[8 / SW];                          // those bytes (D = 256: the half of a key's that has the lane's)
    int pos[CAUSAL ? 8 : 1];                      // positions of the lane's V keys (which are its S^T rows)
};

template <int D, bool CAUSAL>
struct Loader {
    const uint8_t *kc, *ks, *vc, *vs;  // of the sequence and head
    const int32_t* pos;
    int col, grp;

    // `tile` is uniform: the loads take a scalar base, a lane's offset and constants.
    // Slots past `last` read slot `last` (TAIL) or are known to exist.
    template <bool TAIL>
    __device__ __forceinline__ void load(Raw<D, CAUSAL>& r, int tile, int last) const {
        const uint8_t *kb = kc + (int64_t)tile * (D / 2), *ksb = ks + (int64_t)tile * (D / 32);
        const uint8_t *vb = vc + (int64_t)tile * (D / 2), *vsb = vs + (int64_t)tile * (D / 32);
        const int32_t* pb = pos + tile;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t key = 16 * h + col;
            if (TAIL) key = min(key, (uint32_t)(last - tile));
            const uint8_t* p = kb + (key * (D / 2) + grp * (D / 8));
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
            const uint8_t* s = ksb + (key * (D / 32) + (D == 256 ? 2 * grp : grp * (D / 4) / 32));
            if constexpr (D == 256) r.ks[h] = *(const uint16_t*)s;
            else r.ks[h] = *s;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t key = 4 * grp + (16 * (j / 4) + j % 4);
            if (TAIL) key = min(key, (uint32_t)(last - tile));
            const uint8_t* p = vb + (key * (D / 2) + col * (D / 32));
            if constexpr (D == 256) {
                const u32x2 w = *(const u32x2*)p;
                r.v[j][0] = w[0], r.v[j][1] = w[1];
            } else {
                r.v[j][0] = *(const typename Bytes<D / 32>::type*)p;
            }
            // (four keys' scales lie together)
            const uint8_t* s = vsb + (key * (D / 32) + (D == 256 ? (col / 8) * 4 : 0));
            if constexpr (D == 256) {
                r.vs[j] = *(const uint32_t*)s;
            } else if constexpr (TAIL) {
                const uint32_t w = *(const typename Bytes<D / 32>::type*)s;
                constexpr int SW = Raw<D, CAUSAL>::SW;
                r.vs[j / SW] = j % SW ? r.vs[j / SW] | w << (32 / SW * (j % SW)) : w;
            } else if (j % 4 == 0) {
                if constexpr (D == 128) {
                    const u32x4_u w = *(const u32x4_u*)s;
#pragma unroll
                    for (int i = 0; i < 4; ++i) r.vs[j + i] = w[i];
                } else if constexpr (D == 64) {
                    const u32x2_u w = *(const u32x2_u*)s;
                    r.vs[j / 2] = w[0], r.vs[j / 2 + 1] = w[1];
                } else {
                    r.vs[j / 4] = *(const u32_u*)s;
                }
            }
            if constexpr (CAUSAL && !TAIL) {
                if (j % 4 == 0) {
                    const u32x4_u w = *(const u32x4_u*)(pb + key);
#pragma unroll
                    for (int i = 0; i < 4; ++i) r.pos[j + i] = (int)w[i];
                }
            } else if constexpr (CAUSAL) {
                r.pos[j] = pb[key];
            }
        }
    }
    // The byte of vs[] that scales the lane's V values.
    __device__ __forceinline__ int v_byte() const {
        return D == 256 ? (col / 2) & 3 : D == 128 ? col / 4 : D == 64 ? col / 8 : 0;
    }
};

// Few rows (NB blocks of 16): the four waves of a workgroup take every fourth key
// tile of its part of the slots and add up what they have at the end.  CAUSAL hides
// keys in every tile; otherwise only the last, partial tile does, and a tree hides some of the drafted tokens: its
// tiles from the first drafted token on take the masked path, the context's the other.
// Bound by memory: D/2 + D/32 bytes of K and as many of V a slot.  The loop holds
// one tile while the next is loaded (26 registers at D = 128), with a scalar base and
// constant offsets; with the checks for a partial tile inside of it, and the mask as a
// second path, it took 250 registers and spilled.  One token of 32 heads, 8 key
// heads, bf16, caches in turn so that none stays in the last-level cache: 64 sequences of 1024 to
// 4096 slots, D = 128, scores kept for the weights: 47 us, 4.2 TB/s of codes, scales and scores (36 with one
// cache); 32 x 8192 slots at D = 64, 128, 256: 39, 60, 114 us, 3.7, 4.7, 5.0 TB/s (32, 50, 114 with
// one); one sequence of 32768 slots 10 us where the codes' bytes are 6.9: the launch and the first loads.
template <class T, int D, int NB, int MASK>
__global__ void __launch_bounds__(256, 2) attend_kernel(AttendParams p) {
    constexpr bool CAUSAL = MASK == MASK_POSITION, TREE = MASK == MASK_TREE;
    typedef typename T::x8 x8;
    typedef typename T::elem elem;
    constexpr int DT = D / 16;  // 16-row tiles of O^T
    constexpr int QS = D / 32;  // k steps of S^T
    constexpr int WAVES = 4, STEP = TILE * WAVES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int bh = blockIdx.x % p.bh;  // with a multiple of 8, a head's row tiles meet in one XCD's L2
    const int row0 = blockIdx.x / p.bh * (NB * 16);
    const int split = blockIdx.y;
    const int z = bh / (int)p.c.h, h = bh - z * (int)p.c.h;
    const int len = __builtin_amdgcn_readfirstlane(length_of(p.lengths, p.length, z, p.most));
    const int count = p.counts ? max(0, min(p.counts[z], p.t)) : p.t;

    Loader<D, CAUSAL> ld;
    {
        const int64_t c = z * p.c.code_stride[0] + h * p.c.code_stride[1];
        const int64_t s = z * p.c.scale_stride[0] + h * p.c.scale_stride[1];
        ld.kc = p.c.k_codes + c, ld.vc = p.c.v_codes + c;
        ld.ks = p.c.k_scales + s, ld.vs = p.c.v_scales + s;
        ld.pos = p.c.positions + z * p.c.slot_stride[0] + h * p.c.slot_stride[1];
        ld.col = col, ld.grp = grp;
    }

    // this part's slots, a whole number of steps but for the last part's
    const int chunk = ((len + p.splits - 1) / p.splits + STEP - 1) / STEP * STEP;
    const int64_t start64 = (int64_t)chunk * split;
    const int start = (int)(start64 < len ? start64 : len);
    const int end = min(start + chunk, len);
    // whole tiles of this wave (a tree: of the context), and whether the partial one is its own
    const int context = len - count;  // (a tree: the slot of the first drafted token; below 0 it has none)
    const int whole = (TREE ? max(0, min(end, context) - start) : end - start) / TILE;
    const int turns = whole > wave ? (whole - wave + WAVES - 1) / WAVES : 0;
    const bool tail = (end - start) % TILE != 0 && whole % WAVES == wave;

    Raw<D, CAUSAL> cur, next;
    if (turns) ld.template load<false>(cur, start + TILE * wave, 0);

    // Q^T and the rows' positions
    x8 q[NB][QS];
    int qpos[NB];
    const uint32_t* bits[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int row = row0 + 16 * b + col;
        const int tok = row / p.group, head = row - tok * p.group;
        const bool valid = tok < count;  // (row < rows follows)
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
        }
        if (TREE) bits[b] = p.tree + z * p.tree_sz + (int64_t)(valid ? tok : 0) * p.tree_words;
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
    const int vbyte = ld.v_byte();

    // One tile.  MASKED: some of its keys may be hidden from some row, past the end
    // (TAIL) or (causal) of a later position than the row's.
    auto compute = [&](const Raw<D, CAUSAL>& r, int tile, auto tail_) {
        constexpr bool TAIL = decltype(tail_)::value, MASKED = CAUSAL || TAIL;
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
            if constexpr (MASKED) {
                uint32_t seen = 0;
                if constexpr (TREE) seen = tree_mask(bits[b], p.tree_words, tile - context);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int at = 16 * (j / 4) + 4 * grp + j % 4, key = tile + at;
                    const bool hidden = (TAIL && key >= end) || (CAUSAL && r.pos[j] > qpos[b]) || (TREE && !(seen >> at & 1));
                    if (hidden) x[j] = -INFINITY, visible[b] &= ~(1u << j);
                }
            }
            if (p.scores) {
                const int row = row0 + 16 * b + col;
                if (row < p.rows) {
                    float* dst = p.scores + ((int64_t)bh * p.rows + row) * p.most + tile + 4 * grp;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (!TAIL || tile + 16 * (j / 4) + 4 * grp + j % 4 < end) dst[16 * (j / 4) + j % 4] = x[j];
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
        for (int j = 0; j < 8; ++j) {
            constexpr int SW = Raw<D, CAUSAL>::SW;
            sc[j] = scale_bits(r.vs[j / SW], 4 / SW * (j % SW) + vbyte);
        }
        if constexpr (MASKED) {
            uint32_t bad = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (__builtin_amdgcn_classf(sc[j], NAN_OR_INF)) bad |= 1u << j, sc[j] = 0.0f;
            if (__any(bad != 0)) {
                // lane l's O^T values are rows 4 (l / 16) + r of each tile: dims
                // (4 (l / 16) + r) D/16 + d, whose block is that of a lane with col = 4 (l / 16) + r
                for (int b = 0; b < NB; ++b)
                    for (int i = 0; i < 4; ++i) {
                        bool hit = false;
                        for (int g = 0; g < 4; ++g) {
                            const uint32_t vis = __shfl((int)visible[b], 16 * g + col);
                            const uint32_t there = __shfl((int)bad, 16 * g + 4 * grp + i);
                            hit |= (vis & there) != 0;
                        }
#pragma unroll
                        for (int bb = 0; bb < NB; ++bb)
#pragma unroll
                            for (int d = 0; d < DT; ++d)
#pragma unroll
                                for (int ii = 0; ii < 4; ++ii)
                                    if (hit && bb == b && ii == i) acc[bb][d][ii] = __builtin_nanf("");
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

    for (int i = 0; i < turns; ++i) {
        const int tile = start + TILE * (wave + WAVES * i);
        if (i + 1 < turns) ld.template load<false>(next, tile + STEP, 0);
        compute(cur, tile, std::false_type());
        cur = next;
    }
    if constexpr (TREE) {
        for (int i = whole + (wave - whole % WAVES + WAVES) % WAVES; start + TILE * i < end; i += WAVES) {
            ld.template load<true>(cur, start + TILE * i, len - 1);
            compute(cur, start + TILE * i, std::true_type());
        }
    } else if (tail) {
        const int tile = start + TILE * whole;
        ld.template load<true>(cur, tile, len - 1);
        compute(cur, tile, std::true_type());
    }

#pragma unroll
    for (int b = 0; b < NB; ++b) {
        l[b] += __shfl_xor(l[b], 16);
        l[b] += __shfl_xor(l[b], 32);
        // rows past the count are empty (their q was taken as 0)
        if ((row0 + 16 * b + col) / p.group >= count) m[b] = NEVER, l[b] = 0.0f;
    }
    // the waves add up what they have, through LDS: each leaves its sums, scaled to the
    // rows' common maximum, and every thread adds E values of a row
    constexpr int ROWS = NB * 16, E = ROWS * D / 256, PITCH = D + 4;
    __shared__ float2 ml[WAVES][ROWS];
    __shared__ float part[WAVES][ROWS][PITCH];
#pragma unroll
    for (int b = 0; b < NB; ++b)
        if (grp == 0) ml[wave][16 * b + col] = make_float2(m[b], l[b]);
    __syncthreads();
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        float mm = NEVER;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) mm = fmaxf(mm, ml[k][16 * b + col].x);
        const float f = __builtin_amdgcn_exp2f(m[b] - mm);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float* at = &part[wave][16 * b + col][(4 * grp + i) * DT];
#pragma unroll
            for (int d = 0; d < DT; ++d) at[d] = acc[b][d][i] * f;
        }
    }
    __syncthreads();
    const int r = threadIdx.x / (D / E), d0 = threadIdx.x % (D / E) * E;
    const int row = row0 + r;
    if (row >= p.rows) return;
    float mm = NEVER, ll = 0.0f;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) mm = fmaxf(mm, ml[k][r].x);
#pragma unroll
    for (int k = 0; k < WAVES; ++k) ll += ml[k][r].y * __builtin_amdgcn_exp2f(ml[k][r].x - mm);
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = (part[0][r][d0 + e] + part[1][r][d0 + e]) + (part[2][r][d0 + e] + part[3][r][d0 + e]);
    const int64_t at = ((int64_t)split * p.bh + bh) * p.rows + row;
    if (d0 == 0 && p.part_ml) p.part_ml[at] = make_float2(mm, ll);
    if (p.splits > 1) {
        float* dst = p.part_o + at * D + d0;
#pragma unroll
        for (int e = 0; e < E; e += 2) *(float2*)(dst + e) = make_float2(sum[e], sum[e + 1]);
        return;
    }
    // (a NaN sum is a row whose scores are NaN)
    const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
    const int tok = row / p.group, head = row - tok * p.group;
    const int64_t hq = h * p.group + head;
    uint32_t* dst = (uint32_t*)((elem*)p.o + z * p.os[0] + hq * p.os[1] + tok * p.os[2] + d0);
#pragma unroll
    for (int e = 0; e < E; e += 2) dst[e / 2] = ll == 0.0f ? 0u : pack2<T>(sum[e] * inv, sum[e + 1] * inv);
    if (d0 == 0) {
        const float lse2 = ll == 0.0f ? -INFINITY : mm + __builtin_amdgcn_logf(ll);
        if (p.lse) p.lse[(z * (int64_t)p.heads + hq) * p.t + tok] = lse2 * LN2;
        if (p.row_lse) p.row_lse[(int64_t)bh * p.rows + row] = lse2;
    }
}

// Many rows: each of the workgroup's W waves has 32 rows of its own, and all
// share the key tile.  Its codes are converted once per workgroup and kept in LDS as
// the operands of v_mfma_f32_32x32x16 themselves: fragment f is 64 lanes of 16 bytes,
// so that writes and reads are linear.  Of the two buffers one is computed with while
// the next tile is converted into the other, from codes loaded a tile ahead.
//   S^T = K Q^T  A: lane l has the key l % 32 and 8 values a step of the D/2 that
//                start at (l / 32) * D/2, so a fragment is one dword of codes.
//   O^T = V^T P^T  S^T leaves lane l the row l % 32 and the keys 8 a + 4 (l / 32) + b;
//                step s takes k = 8 (l / 32) + j as key 16 s + 8 (j / 4) + 4 (l / 32) + j % 4.
//                A: lane l has these keys of the value (l % 32) * D/32 + t in fragment t.
// With eight waves a tile is computed with in two pieces; half of the waves convert their
// part of the next tile before the first piece, half after it, so that the two waves of a SIMD
// want the matrix unit at different times.
// Bound by the matrix and the vector units together: a chunk of 2048 tokens, 32 heads,
// over 16384 slots of 8 key heads, D = 128, bf16, causal: 468 to 478 us, 1080 to 1100 TFLOP/s; at D = 64
// 326 us, 790 TFLOP/s, where the vector unit is busy for 56 % of it and the matrix unit for 31 (45 and 45 at
// D = 128).  (Four waves, which convert twice as often: 75 us more; eight that convert together: 3, and of calls for
// 1024 tokens with weights at D = 64, two sequences of 32 heads, 8192 slots of 8, 290 against 280, at D = 256, 16
// heads, 16384 slots of 4, 494 against 459.  The two
// pieces in a loop instead of code of their own: 40 us more.  Direct operands
// without LDS, 32 rows a wave: 1107.  Halves of a tile whose softmax and products alternate,
// raised wave priority around the products, LDS reads two to eight MFMAs ahead:
// no gain with four waves.)
// With G = 2 the waves w and w + W / 2 have the same rows and a half of each tile's keys each, and add up at the end.
template <int D, int W, int G = 1>
struct Many {
    static constexpr int KEYS = (D == 256 ? 8 : 16) * W; // of a tile: its fragments take 8 KB a wave at D = 128, 256
    static constexpr int PIECE = G > 1 ? KEYS / G : D == 256 ? 32 : 64;  // keys between two looks at the running maximum
    static constexpr int PIECES = G > 1 ? 1 : W / 4;     // of a tile, that a wave computes with
    static constexpr int KF = KEYS / 32 * (D / 16) / W;  // K fragments a wave converts
    static constexpr int VF = KEYS / 16 * (D / 32) / W;  // V fragments
    static constexpr int KFRAGS = W * KF, FRAGS = W * (KF + VF);
    static constexpr int PER_BLOCK = W / (KEYS / 32);    // waves that share a block of 32 keys' K
    static constexpr int ROWS = 32 * W / G;
};

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(F16::x8 a, F16::x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(BF16::x8 a, BF16::x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

template <class T, int D, int MASK, int W, int G = 1>
__global__ void __launch_bounds__(64 * W, 2) attend_many_kernel(AttendParams p) {
    constexpr bool CAUSAL = MASK == MASK_POSITION, TREE = MASK == MASK_TREE;
    typedef Many<D, W, G> M;
    typedef typename T::x8 x8;
    typedef typename T::elem elem;
    constexpr int QS = D / 16, DT = D / 32, KEYS = M::KEYS, PIECE = M::PIECE, SB = PIECE / 32;
    __shared__ u32x4 frag[2][M::FRAGS][64];
    __shared__ int kpos[2][CAUSAL ? KEYS : 1];
    __shared__ int spoiled[2][W];  // a wave's V codes of the tile hold a NaN block
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int bh = blockIdx.x % p.bh;  // with a multiple of 8, a head's row tiles meet in one XCD's L2
    const int z = bh / (int)p.c.h, h = bh - z * (int)p.c.h;
    const int len = __builtin_amdgcn_readfirstlane(length_of(p.lengths, p.length, z, p.most));
    const int count = p.counts ? max(0, min(p.counts[z], p.t)) : p.t;
    const int part = wave / (W / G);  // of a tile's keys, the wave's own (G > 1)
    const int row = blockIdx.x / p.bh * M::ROWS + 32 * (G > 1 ? wave % (W / G) : wave) + col;
    const int tok = row / p.group, head = row - tok * p.group;
    const bool valid = tok < count;  // (row < rows follows)
    const int64_t cb = z * p.c.code_stride[0] + h * p.c.code_stride[1];
    const int64_t sb = z * p.c.scale_stride[0] + h * p.c.scale_stride[1];
    const uint8_t *kc = p.c.k_codes + cb, *vc = p.c.v_codes + cb, *ks = p.c.k_scales + sb, *vs = p.c.v_scales + sb;
    const int32_t* pos = p.c.positions + z * p.c.slot_stride[0] + h * p.c.slot_stride[1];

    const int chunk = ((len + p.splits - 1) / p.splits + KEYS - 1) / KEYS * KEYS;
    const int64_t start64 = (int64_t)chunk * blockIdx.y;
    const int start = (int)(start64 < len ? start64 : len);
    const int end = min(start + chunk, len);

    // Q^T
    x8 q[QS];
    int qpos = -0x7fffffff - 1, least = 0x7fffffff, greatest = -0x7fffffff - 1;
    {
        u32x4 w[QS] = {};
        if (valid) {
            const elem* src = (const elem*)p.q + z * p.qs[0] + (int64_t)(h * p.group + head) * p.qs[1] + tok * p.qs[2] + half * (D / 2);
#pragma unroll
            for (int i = 0; i < QS; ++i) w[i] = *(const u32x4*)(src + 8 * i);
        }
#pragma unroll
        for (int i = 0; i < QS; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[i][j] ^= p.neg;
            q[i] = __builtin_bit_cast(x8, w[i]);
        }
        if (CAUSAL) {
            const int64_t at = (p.pos_start ? (int64_t)p.pos_start[z] : (int64_t)len - count) + tok;
            if (valid) least = greatest = qpos = (int)(at > 0x7fffffff ? 0x7fffffff : at);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                least = min(least, __shfl_xor(least, d));
                greatest = max(greatest, __shfl_xor(greatest, d));
            }
        }
    }

    const int context = len - count;  // (a tree: the slot of the first drafted token)
    const uint32_t* const bits = TREE ? p.tree + z * p.tree_sz + (int64_t)(valid ? tok : 0) * p.tree_words : nullptr;

    // this wave's part of a tile's conversion
    struct {
        uint32_t k[M::KF], ks;
        uint32_t v[8], vs[8];
        int pos;
    } raw;
    const int kblock = wave / M::PER_BLOCK, kpart = wave % M::PER_BLOCK;
    const int vstep = D == 256 ? wave / 2 : wave, vpart = D == 256 ? wave % 2 : 0;
    // V codes of a lane: D/64 bytes of a key (D = 256: of its half of them; D = 32: half a byte)
    const uint32_t koff = half * (D / 4) + kpart * (4 * M::KF);
    const uint32_t ksoff = (half * (D / 2) + kpart * (8 * M::KF)) / 32;
    const uint32_t voff = D == 32 ? col / 2 : D == 256 ? col * 4 + vpart * 2 : col * (D / 64);
    const uint32_t vsoff = D == 256 ? (col / 16) * 4 : 0;
    const int vbyte = D == 256 ? (col / 4) & 3 : D == 128 ? col / 8 : D == 64 ? col / 16 : 0;
    auto load_tile = [&](int tile, auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        // keys past the length repeat the last (without a check the addresses are constants apart)
        const uint32_t last = len - 1 - tile;
        auto inside = [&](uint32_t key) { return WHOLE ? key : min(key, last); };
        const uint8_t* kb = kc + (int64_t)tile * (D / 2);
        const uint8_t* vb = vc + (int64_t)tile * (D / 2);
        {
            const uint32_t key = inside(32 * kblock + col);
            const uint8_t* src = kb + (key * (D / 2) + koff);
            if constexpr (M::KF == 4) {
                const u32x4 w = *(const u32x4*)src;
#pragma unroll
                for (int i = 0; i < 4; ++i) raw.k[i] = w[i];
            } else if constexpr (M::KF == 2) {
                const u32x2 w = *(const u32x2*)src;
                raw.k[0] = w[0], raw.k[1] = w[1];
            } else {
                raw.k[0] = *(const uint32_t*)src;
            }
            raw.ks = (ks + (int64_t)tile * (D / 32))[key * (D / 32) + ksoff];
        }
        const uint8_t* vsb = vs + (int64_t)tile * (D / 32);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t key = inside(16 * vstep + 4 * half + (8 * (j / 4) + j % 4));
            const uint8_t* src = vb + (key * (D / 2) + voff);
            if constexpr (D >= 128) raw.v[j] = *(const uint16_t*)src;
            else raw.v[j] = *src;
            const uint8_t* s = vsb + (key * (D / 32) + vsoff);
            if constexpr (D == 128 && WHOLE) {
                if (j % 4 == 0) {  // four keys' scales lie together
                    const u32x4_u w = *(const u32x4_u*)s;
#pragma unroll
                    for (int i = 0; i < 4; ++i) raw.vs[j + i] = w[i];
                }
            } else {
                raw.vs[j] = *(const typename Bytes<D == 256 ? 4 : D / 32>::type*)s;
            }
        }
        if (CAUSAL && threadIdx.x < KEYS) raw.pos = pos[tile + inside(threadIdx.x)];
    };
    auto load = [&](int tile) {
        // (at D = 256 the second path's registers spill: 256 rows of 32 x 8192 slots 113 -> 259 us; one wave a
        // SIMD instead of two, without spills: 158)
        if (D != 256 && tile + KEYS <= len) load_tile(tile, std::true_type());
        else load_tile(tile, std::false_type());
    };
    auto convert = [&](int buf) {
        const float ksc = scale_bits(raw.ks, 0);
#pragma unroll
        for (int i = 0; i < M::KF; ++i) {
            const uint32_t w = raw.k[i];
            frag[buf][wave * M::KF + i][lane] = (u32x4){T::template cvt<0>(w, ksc), T::template cvt<1>(w, ksc),
                                                         T::template cvt<2>(w, ksc), T::template cvt<3>(w, ksc)};
        }
        // a NaN block of V is converted as 0, and noted: it must reach only rows that see its key
        float sc[8];
        bool bad = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sc[j] = scale_bits(raw.vs[j], vbyte);
            bad |= __builtin_amdgcn_classf(sc[j], NAN_OR_INF);
        }
        const bool any = __any(bad);
        if (__builtin_expect(any, 0)) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (__builtin_amdgcn_classf(sc[j], NAN_OR_INF)) sc[j] = 0.0f;
        }
        if (lane == 0) spoiled[buf][wave] = any;
#pragma unroll
        for (int pr = 0; pr < (M::VF + 1) / 2; ++pr) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = pr == 0 ? T::template cvt<0>(raw.v[j], sc[j]) : T::template cvt<1>(raw.v[j], sc[j]);
            const uint32_t lo = D == 32 && (col & 1) ? 0x07060302u : 0x05040100u;
            u32x4 even, odd;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                even[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], lo);
                odd[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x07060302u);
            }
            frag[buf][M::KFRAGS + wave * M::VF + 2 * pr][lane] = even;
            if (M::VF > 1) frag[buf][M::KFRAGS + wave * M::VF + 2 * pr + 1][lane] = odd;
        }
        if (CAUSAL && threadIdx.x < KEYS) kpos[buf][threadIdx.x] = raw.pos;
    };

    f32x16 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;
    float m = NEVER, l = 0.0f;

    auto compute = [&](int buf, int tile, int piece) {
        const int kb = piece * SB, vb = M::KFRAGS + piece * 2 * SB * DT, at = piece * PIECE;
        tile += at;
        bool masked = tile + PIECE > (TREE ? min(end, context) : end);
        if (CAUSAL) {
            const int kp = kpos[buf][at + (lane & (PIECE - 1))];
            masked |= __any(kp > least);
            if (!__any(kp <= greatest)) return;
        }
        f32x16 s[SB];
#pragma unroll
        for (int b = 0; b < SB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[b][r] = 0.0f;
#pragma unroll
        for (int i = 0; i < QS; ++i)
#pragma unroll
            for (int b = 0; b < SB; ++b) s[b] = mfma32(__builtin_bit_cast(x8, frag[buf][(kb + b) * QS + i][lane]), q[i], s[b]);
        if (__builtin_expect(masked, 0)) {
#pragma unroll
            for (int b = 0; b < SB; ++b) {
                const uint32_t seen = TREE ? tree_mask(bits, p.tree_words, tile + 32 * b - context) : 0u;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int sub = 8 * (r / 4) + 4 * half + r % 4, key = 32 * b + sub;
                    bool hidden = tile + key >= end;
                    if (CAUSAL) hidden |= kpos[buf][at + key] > qpos;
                    if (TREE) hidden |= !(seen >> sub & 1);
                    if (hidden) s[b][r] = -INFINITY;
                }
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < SB; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
        top *= p.scale;
        if (__any(top > m + SLACK)) {
            top = fmaxf(top, __shfl_xor(top, 32));
            const float now = fmaxf(m, top);
            const float f = __builtin_amdgcn_exp2f(m - now);
            m = now;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d] *= f;
        }
        x8 pb[2 * SB];
#pragma unroll
        for (int b = 0; b < SB; ++b)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][8 * t + j], p.scale, -m));
                l += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
                pb[2 * b + t] = __builtin_bit_cast(x8, (u32x4){pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7])});
            }
#pragma unroll
        for (int k = 0; k < 2 * SB; ++k)
#pragma unroll
            for (int d = 0; d < DT; ++d)
                acc[d] = mfma32(__builtin_bit_cast(x8, frag[buf][vb + k * DT + d][lane]), pb[k], acc[d]);
        int nan = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) nan |= spoiled[buf][w];
        if (__builtin_expect(nan, 0)) {
            // NaN blocks of V, into the rows that see them: register r holds the values
            // D/32 (8 (r / 4) + 4 half + r % 4) + d, which lie in one block
            uint32_t hit = 0;
            for (int k = 0; k < PIECE && tile + k < end; ++k) {
                bool sees = true;
                if (CAUSAL) sees = kpos[buf][at + k] <= qpos;
                if (TREE) sees = tree_mask(bits, p.tree_words, tile + k - context) & 1;
                if (!sees) continue;
                for (int r = 0; r < 16; ++r) {
                    const int i = 8 * (r / 4) + 4 * half + r % 4;
                    if (vs[(int64_t)(tile + k) * (D / 32) + i * D / 1024] == 255) hit |= 1u << r;
                }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (hit & (1u << r))
#pragma unroll
                    for (int d = 0; d < DT; ++d) acc[d][r] = __builtin_nanf("");
        }
    };

    const bool late = W > 4 && wave >= 4;
    if (start < end) {
        load(start);
        convert(0);
        if (start + KEYS < end) load(start + KEYS);
        int buf = 0;
        for (int tile = start; tile < end; tile += KEYS, buf ^= 1) {
            __syncthreads();  // this tile is in LDS, and nobody reads the other buffer any more
            const int mine = G > 1 ? part : 0;
            const bool there = G == 1 || tile + mine * PIECE < end;
            if (late && there) compute(buf, tile, mine);
            if (tile + KEYS < end) convert(buf ^ 1);
            if (tile + 2 * KEYS < end) load(tile + 2 * KEYS);
            if (!late && there) compute(buf, tile, mine);
#pragma unroll
            for (int i = 1; i < M::PIECES; ++i)
                if (tile + i * PIECE < end) compute(buf, tile, i);
        }
    }
    l += __shfl_xor(l, 32);
    if (!valid) m = NEVER, l = 0.0f;  // past the count (q was taken as 0)
    if constexpr (G > 1) {
        // the waves of a row add up their parts of the keys, through the tiles' LDS
        constexpr int RW = W / G;
        static_assert(sizeof(frag) >= (W - RW) * 64 * DT * 64, "the sums fit the tiles' LDS");
        f32x4* const sums = (f32x4*)&frag[0][0][0];  // [wave - RW][DT * 4][64]
        __shared__ float2 ml[(W - RW) * 64];
        __syncthreads();
        if (part) {
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int a = 0; a < 4; ++a)
                    sums[((wave - RW) * DT * 4 + d * 4 + a) * 64 + lane] = (f32x4){acc[d][4 * a], acc[d][4 * a + 1], acc[d][4 * a + 2], acc[d][4 * a + 3]};
            ml[(wave - RW) * 64 + lane] = make_float2(m, l);
        }
        __syncthreads();
        if (part) return;
#pragma unroll
        for (int g = 0; g < G - 1; ++g) {
            const float2 v = ml[(g * RW + wave) * 64 + lane];
            const float now = fmaxf(m, v.x);
            const float f = __builtin_amdgcn_exp2f(m - now), x = __builtin_amdgcn_exp2f(v.x - now);
            m = now;
            l = l * f + v.y * x;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const f32x4 o = sums[((g * RW + wave) * DT * 4 + d * 4 + a) * 64 + lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[d][4 * a + e] = acc[d][4 * a + e] * f + o[e] * x;
                }
        }
    }
    if (row >= p.rows) return;
    if (p.splits > 1) {
        const int64_t at = ((int64_t)blockIdx.y * p.bh + bh) * p.rows + row;
        if (half == 0) p.part_ml[at] = make_float2(m, l);
        float* dst = p.part_o + at * D;
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int d = 0; d < DT; ++d) dst[(8 * (r / 4) + 4 * half + r % 4) * DT + d] = acc[d][r];
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t hq = h * p.group + head;
    elem* dst = (elem*)p.o + z * p.os[0] + hq * p.os[1] + tok * p.os[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        elem* at = dst + (8 * (r / 4) + 4 * half + r % 4) * DT;
        if constexpr (DT == 1) {
            *at = (elem)(l == 0.0f ? 0.0f : acc[0][r] * inv);
        } else {
#pragma unroll
            for (int d = 0; d < DT; d += 2)
                ((uint32_t*)at)[d / 2] = l == 0.0f ? 0u : pack2<T>(acc[d][r] * inv, acc[d + 1][r] * inv);
        }
    }
    if (half == 0) {
        const float lse2 = l == 0.0f ? -INFINITY : m + __builtin_amdgcn_logf(l);
        if (p.lse) p.lse[(z * (int64_t)p.heads + hq) * p.t + tok] = lse2 * LN2;
        if (p.row_lse) p.row_lse[(int64_t)bh * p.rows + row] = lse2;
    }
}

// Sum of a row's parts: D / 4 lanes hold a row, four values each, and `pp` such
// groups of a workgroup take every pp-th part of it, so that the loads of a row's
// parts do not wait for each other (64 parts of 32 rows: 3.9 us, one after another 41).
template <class T, int D>
__device__ __forceinline__ void join_rows(const AttendParams& p, int pp, int block) {
    constexpr int G = D / 4, GROUPS = 256 / G;
    __shared__ f32x4 part[256];
    __shared__ float2 ml[GROUPS];
    const int lane = threadIdx.x % G, grp = threadIdx.x / G;
    const int64_t all = (int64_t)p.bh * p.rows;
    const int64_t id = (int64_t)block * (GROUPS / pp) + grp / pp;  // bh * rows + row
    float m = NEVER, l = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    if (id < all) {
        constexpr int U = 8;  // parts whose loads are under way together
        for (int s0 = grp % pp; s0 < p.splits; s0 += U * pp) {
            float2 v[U];
            f32x4 x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int s = min(s0 + u * pp, p.splits - 1);
                v[u] = p.part_ml[s * all + id];
                x[u] = *(const f32x4*)(p.part_o + (s * all + id) * D + 4 * lane);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (s0 + u * pp >= p.splits || v[u].y == 0.0f) continue;  // (0: no slot in this part)
                const float now = fmaxf(m, v[u].x);
                const float f = __builtin_amdgcn_exp2f(m - now), g = __builtin_amdgcn_exp2f(v[u].x - now);
                m = now;
                l = l * f + v[u].y * g;
                o = o * f + x[u] * g;
            }
        }
    }
    if (pp > 1) {
        part[threadIdx.x] = o;
        if (lane == 0) ml[grp] = make_float2(m, l);
        __syncthreads();
        if (grp % pp != 0 || id >= all) return;
        for (int i = 1; i < pp; ++i) {
            const float2 v = ml[grp + i];
            if (v.y == 0.0f) continue;
            const float now = fmaxf(m, v.x);
            const float f = __builtin_amdgcn_exp2f(m - now), g = __builtin_amdgcn_exp2f(v.x - now);
            m = now;
            l = l * f + v.y * g;
            o = o * f + part[threadIdx.x + i * G] * g;
        }
    } else if (id >= all) {
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int bh = (int)(id / p.rows), row = (int)(id - (int64_t)bh * p.rows);
    const int z = bh / (int)p.c.h, h = bh - z * (int)p.c.h;
    const int tok = row / p.group, head = row - tok * p.group;
    const int64_t hq = h * p.group + head;
    typename T::elem* dst = (typename T::elem*)p.o + z * p.os[0] + hq * p.os[1] + tok * p.os[2] + 4 * lane;
    *(u32x2*)dst = (u32x2){pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
    if (lane == 0) {
        const float lse2 = l == 0.0f ? -INFINITY : m + __builtin_amdgcn_logf(l);
        if (p.lse) p.lse[(z * (int64_t)p.heads + hq) * p.t + tok] = lse2 * LN2;
        if (p.row_lse) p.row_lse[id] = lse2;
    }
}

// Weights of up to 32 rows, from their scores and their parts' sums; a thread takes
// four slots, a workgroup 1024.
__device__ __forceinline__ void add_weights(const AttendParams& p, int block) {
    __shared__ float sums[32];
    const int bh = block % p.bh;
    const int z = bh / (int)p.c.h, h = bh - z * (int)p.c.h;
    const int len = length_of(p.lengths, p.length, z, p.most);
    const int count = p.counts ? max(0, min(p.counts[z], p.t)) : p.t;
    const int rows = count * p.group;
    const int64_t first = (int64_t)(block / p.bh) * 1024;
    if (first >= len) return;
    {
        // eight lanes a row: log2 of its sum
        const int row = threadIdx.x / 8;
        const int64_t all = (int64_t)p.bh * p.rows, id = (int64_t)bh * p.rows + row;
        float m = NEVER, l = 0.0f;
        if (row < rows) {
            for (int s = threadIdx.x % 8; s < p.splits; s += 8) {
                const float2 v = p.part_ml[s * all + id];
                if (v.y == 0.0f) continue;
                const float now = fmaxf(m, v.x);
                l = l * __builtin_amdgcn_exp2f(m - now) + v.y * __builtin_amdgcn_exp2f(v.x - now);
                m = now;
            }
        }
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) {
            const float m2 = __shfl_xor(m, d), l2 = __shfl_xor(l, d);
            const float now = fmaxf(m, m2);
            l = l * __builtin_amdgcn_exp2f(m - now) + l2 * __builtin_amdgcn_exp2f(m2 - now);
            m = now;
        }
        if (threadIdx.x % 8 == 0) sums[row] = l == 0.0f ? -INFINITY : m + __builtin_amdgcn_logf(l);
    }
    __syncthreads();
    const int64_t slot = first + 4 * threadIdx.x;
    if (slot >= len) return;
    float* w = p.c.weights + z * p.c.slot_stride[0] + h * p.c.slot_stride[1] + slot;
    const float* x = p.scores + (int64_t)bh * p.rows * p.most + slot;
    // a slot that the row does not see has a score of -inf (and a row that sees none: in all)
    auto weight = [](float s, float sum) { return s == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s - sum); };
    if (slot + 4 <= len) {
        f32x4 sum = {0, 0, 0, 0};
#pragma unroll 4
        for (int r = 0; r < rows; ++r) {
            const f32x4 s = *(const f32x4_u*)(x + (int64_t)r * p.most);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] += weight(s[i], sums[r]);
        }
        *(f32x4_u*)w = *(const f32x4_u*)w + sum;
    } else {
        for (int i = 0; slot + i < len; ++i) {
            float sum = 0.0f;
            for (int r = 0; r < rows; ++r) sum += weight(x[(int64_t)r * p.most + i], sums[r]);
            w[i] += sum;
        }
    }
}

// What follows attend_kernel or attend_many_kernel: the first join_blocks workgroups
// join parts, the others add weights.
template <class T, int D>
__global__ void __launch_bounds__(256) finish_kernel(AttendParams p, int pp, int join_blocks) {
    if ((int)blockIdx.x < join_blocks) join_rows<T, D>(p, pp, blockIdx.x);
    else add_weights(p, blockIdx.x - join_blocks);
}

// Weights of many rows: the scores are computed again, now that the rows' sums are
// known.  Each wave holds 32 keys of its own as operands of the 32 x 32 MFMA (32
// registers at D = 128, 64 at 256); blocks of 32 rows of Q pass by in LDS, as operands
// too, two buffers of ROW_BLOCKS blocks.  A workgroup takes the groups of row blocks
// blockIdx.y, blockIdx.y + gridDim.y, ...
// Bound as attend_many_kernel is, with half its products and all of its exponentials: 295 to 316
// us for the chunk above, of which no part stands alone (in copies without it: loads of Q 56 less, seven of
// eight products 94, exponentials 38).  Up to D = 128 a wave keeps to 128 registers, so
// that four waves of a SIMD hide each other's products and exponentials; with 64
// keys, two waves: 24 us more.  Row blocks between barriers, one, two, three, four: the two
// kernels 861, 843, 840, 848 at D = 128, 346, 336, 329, 329 at D = 64.  D = 256 (1024 tokens of
// 16 heads, 16384 slots of 4) does not fit four waves: 536 us spilled, 513 with two; one row block
// 548, two 514, four, which leave room for one workgroup, 666.  (16 x 16 tiles with Q from
// global memory: 492 of the chunk.)
template <int D>
struct Weigh {
    static constexpr int KEYS = 32;  // of a wave
    static constexpr int WAVES = D == 256 ? 4 : 8;
    static constexpr int OCCUPANCY = D == 256 ? 2 : 4;  // waves of a SIMD
    static constexpr int ROW_BLOCKS = D == 256 ? 2 : 3;
    static constexpr int WG_KEYS = WAVES * KEYS;
};

template <class T, int D, bool CAUSAL>
__global__ void __launch_bounds__(64 * Weigh<D>::WAVES, Weigh<D>::OCCUPANCY) weights_kernel(AttendParams p) {
    typedef typename T::x8 x8;
    typedef typename T::elem elem;
    constexpr int QS = D / 16, KEYS = Weigh<D>::KEYS;
    constexpr int WAVES = Weigh<D>::WAVES, QF = (QS + WAVES - 1) / WAVES;  // fragments of Q a wave brings
    constexpr int RB = Weigh<D>::ROW_BLOCKS;
    __shared__ u32x4 frag[2][RB][QS][64];
    __shared__ int kpos[CAUSAL ? WAVES * KEYS : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int bh = blockIdx.x % p.bh;
    const int z = bh / (int)p.c.h, h = bh - z * (int)p.c.h;
    const int len = __builtin_amdgcn_readfirstlane(length_of(p.lengths, p.length, z, p.most));
    const int count = p.counts ? max(0, min(p.counts[z], p.t)) : p.t;
    const int rows = count * p.group;
    const int64_t wg_tile = (int64_t)(blockIdx.x / p.bh) * Weigh<D>::WG_KEYS;
    if (wg_tile >= len) return;
    const int tile = (int)wg_tile + KEYS * wave;  // (may lie past the length: its keys repeat the last)
    const uint8_t* kc = p.c.k_codes + z * p.c.code_stride[0] + h * p.c.code_stride[1];
    const uint8_t* ks = p.c.k_scales + z * p.c.scale_stride[0] + h * p.c.scale_stride[1];
    const int32_t* pos = p.c.positions + z * p.c.slot_stride[0] + h * p.c.slot_stride[1];
    int far = -0x7fffffff - 1, near = 0x7fffffff;  // positions of the wave's keys
    if (CAUSAL) {
        const int v = pos[min(tile + (lane & (KEYS - 1)), len - 1)];
        kpos[KEYS * wave + (lane & (KEYS - 1))] = v;
        far = near = v;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            far = max(far, __shfl_xor(far, d));
            near = min(near, __shfl_xor(near, d));
        }
        far = __builtin_amdgcn_readfirstlane(far);
        near = __builtin_amdgcn_readfirstlane(near);
    }
    x8 k[QS];
    {
        const int key = min(tile + col, len - 1);
        const uint8_t* src = kc + (int64_t)key * (D / 2) + half * (D / 4);
        const uint8_t* s = ks + (int64_t)key * (D / 32);
#pragma unroll
        for (int i = 0; i < QS; ++i) {
            const uint32_t w = *(const uint32_t*)(src + 4 * i);
            const float sc = scale_bits(s[(half * (D / 2) + 8 * i) / 32], 0);
            const u32x4 kv = {T::template cvt<0>(w, sc), T::template cvt<1>(w, sc), T::template cvt<2>(w, sc),
                              T::template cvt<3>(w, sc)};
            k[i] = __builtin_bit_cast(x8, kv);
        }
    }
    const int64_t first = CAUSAL ? (p.pos_start ? (int64_t)p.pos_start[z] : (int64_t)len - count) : 0;
    const elem* qb = (const elem*)p.q + z * p.qs[0] + (int64_t)h * p.group * p.qs[1];
    const float* lse = p.row_lse + (int64_t)bh * p.rows;
    const float scale = p.neg ? -p.scale : p.scale;
    u32x4 raw[RB][QF];
    float lse_next[RB];
    int tok_next[RB];
    // the row of a lane in the next block to be loaded, as token and head of the group
    const int step = 32 * RB * gridDim.y;
    const int more_tok = 32 / p.group, more_head = 32 - more_tok * p.group;  // a block of rows further
    const int step_tok = (step - 32 * (RB - 1)) / p.group, step_head = step - 32 * (RB - 1) - step_tok * p.group;
    int tok = (32 * RB * (int)blockIdx.y + col) / p.group, head = 32 * RB * (int)blockIdx.y + col - tok * p.group;
    auto load = [&](int row0) {
#pragma unroll
        for (int g = 0; g < RB; ++g) {
            const int row = row0 + 32 * g + col;
            tok_next[g] = min(tok, count - 1);
            const elem* src = qb + head * p.qs[1] + tok_next[g] * p.qs[2] + half * (D / 2);
#pragma unroll
            for (int i = 0; i < QF; ++i)
                if (QS >= WAVES || wave < QS) raw[g][i] = *(const u32x4*)(src + 8 * (wave * QF + i));
            lse_next[g] = lse[min(row, rows - 1)];
            tok += g < RB - 1 ? more_tok : step_tok;
            head += g < RB - 1 ? more_head : step_head;
            if (head >= p.group) head -= p.group, ++tok;
        }
    };
    float lse2[RB];
    int tok2[RB];
    // (what was loaded is first looked at here: a comparison where it is loaded waits for it, 462 us against 433
    // for 1024 tokens of 16 heads, 16384 slots of 4, at D = 256)
    auto store = [&](int buf, int row0) {
#pragma unroll
        for (int g = 0; g < RB; ++g) {
            // rows past the last and rows that see no slot are hidden below
            lse2[g] = row0 + 32 * g + col < rows && lse_next[g] != -INFINITY ? lse_next[g] : INFINITY;
            tok2[g] = tok_next[g];
#pragma unroll
            for (int i = 0; i < QF; ++i)
                if (QS >= WAVES || wave < QS) frag[buf][g][wave * QF + i][lane] = raw[g][i];
        }
    };
    float sum[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) sum[r] = 0.0f;

    int row0 = 32 * RB * blockIdx.y;
    if (row0 < rows) {
        load(row0);
        store(0, row0);
        if (row0 + step < rows) load(row0 + step);
        int buf = 0;
        for (; row0 < rows; row0 += step, buf ^= 1) {
            __syncthreads();
            float lse_now[RB];
            int tok_now[RB];
#pragma unroll
            for (int g = 0; g < RB; ++g) lse_now[g] = lse2[g], tok_now[g] = tok2[g];
            if (row0 + step < rows) store(buf ^ 1, row0 + step);
            if (row0 + 2 * step < rows) load(row0 + 2 * step);
#pragma unroll
            for (int g = 0; g < RB; ++g) {
                if (row0 + 32 * g >= rows) break;
                bool masked = __any(lse_now[g] == INFINITY);
                int qpos = 0;
                if (CAUSAL) {
                    // the block's rows have positions that grow with the row
                    const int64_t lo = first + __builtin_amdgcn_readfirstlane(tok_now[g]);
                    const int64_t hi = first + __builtin_amdgcn_readlane(tok_now[g], 31);
                    if (near > hi) continue;
                    masked |= far > lo;
                    const int64_t at = first + tok_now[g];
                    qpos = (int)(at > 0x7fffffff ? 0x7fffffff : at);
                }
                f32x16 s;
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
                for (int i = 0; i < QS; ++i) s = mfma32(k[i], __builtin_bit_cast(x8, frag[buf][g][i][lane]), s);
                if (__builtin_expect(masked, 0)) {
                    // (chosen after the exponential: a row whose sum is NaN adds nothing to slots it does not see)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        bool hidden = lse_now[g] == INFINITY;
                        if (CAUSAL) hidden |= kpos[KEYS * wave + 8 * (r / 4) + 4 * half + r % 4] > qpos;
                        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], scale, -lse_now[g]));
                        sum[r] += hidden ? 0.0f : x;
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        sum[r] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], scale, -lse_now[g]));
                }
            }
        }
    }
    float* out = p.part_w ? p.part_w + ((int64_t)blockIdx.y * p.bh + bh) * p.most
                          : p.c.weights + z * p.c.slot_stride[0] + h * p.c.slot_stride[1];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        float v = sum[r];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) v += __shfl_xor(v, d);
        const int key = tile + 8 * (r / 4) + 4 * half + r % 4;
        if (col == 0 && key < len) {
            if (p.part_w) out[key] = v;
            else out[key] += v;
        }
    }
}

// The sums of weights_kernel's parts, where the rows were split.
__global__ void __launch_bounds__(256) join_weights_kernel(AttendParams p, int parts) {
    const int bh = blockIdx.x % p.bh;
    const int z = bh / (int)p.c.h, h = bh - z * (int)p.c.h;
    const int64_t slot = (int64_t)(blockIdx.x / p.bh) * 256 + threadIdx.x;
    if (slot >= length_of(p.lengths, p.length, z, p.most)) return;
    float v = 0.0f;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) v += p.part_w[((int64_t)i * p.bh + bh) * p.most + slot];
    p.c.weights[z * p.c.slot_stride[0] + h * p.c.slot_stride[1] + slot] += v;
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
struct Plan {
    bool few;          // attend_kernel, with nb blocks of 16 rows
    int nb;
    int waves, tiles, splits;
    int groups;        // attend_many_kernel: parts of a tile's keys
    bool scores;       // weights from stored scores
    int weight_tiles, weight_parts;
    uint64_t part_w;
    uint64_t part_o, part_ml, scores_at, row_lse, bytes;  // offsets into the workspace
};

Plan make_plan(const rsfa_cache4_attend_args* a, int cus, bool tree) {
    Plan p{};
    const int64_t group = a->heads / a->cache.h, rows = group * a->t;
    const int64_t bh = a->cache.z * a->cache.h;
    const int64_t most = a->max_length > 0 && a->max_length < a->cache.capacity ? a->max_length : a->cache.capacity;
    // (32 key heads of 8192 slots, bf16, causal, caches in turn, few and many rows' kernel at D = 64, 128, 256: 32 rows 17
    // and 26 us, 20 and 29, 38 and 55; 64 rows 24 and 27, 32 and 31, 63 and 66; 128 rows 36 and 31, 53 and 37, 94 and 92:
    // up to 64 rows the few rows' kernel would still be ahead at D = 64 and 256)
    // A tree's rows stay with it for longer: 8 or 16 sequences of 8 key heads, D = 64 and 128, 4096 and 8192 slots, bf16, caches in
    // turn, 48 and 64 rows 25 and 35 us, 33 and 37, with many rows' kernel 49 and 35, 66 and 68 (its waves in two groups,
    // below, 35, 47, 49); 32 sequences of up to 4096 slots, 100 rows, 86, 111 and 76; D = 256, 8000 slots, 120 rows 45, 58 and 53.
    const bool few = rows <= (tree ? a->cache.head_dim == 256 ? 128 : 64 : 32);
    p.few = few;
    p.nb = rows <= 16 || a->cache.head_dim == 256 ? 1 : 2;
    // (D = 256, four and eight waves: 128 rows of the same 92 and 96 us, 192 rows 115 and 107; below 256 they are
    // the same within half a microsecond)
    p.waves = few || (a->cache.head_dim == 256 && rows <= 128) ? 4 : 8;
    // Up to 128 rows leave half of the eight waves without rows of their own: these take half of the others' keys.
    // (Without a tree they idle, as they always have: sums in another order would be other bits.)
    p.groups = tree && !few && rows <= 128 ? 2 : 1;
    const int64_t tile_rows = few ? 16 * p.nb : 32 * p.waves / p.groups;
    p.tiles = (int)((rows + tile_rows - 1) / tile_rows);
    // Enough workgroups for the chip, of at least four steps each.  Few rows: eight
    // workgroups a CU even out lengths (64 sequences of 1024 to 4096 slots 46.6 -> 44.9 us
    // against four); fewer steps each cost more in joining them (one sequence of
    // 32768 slots: 13.1, 16.4 with two steps each, 22.9 with one).
    const int64_t step = few ? 4 * TILE : 16 * p.waves;
    const int64_t full = (few ? 8 : 8 / p.waves) * (int64_t)cus;
    int64_t want = (full + bh * p.tiles - 1) / (bh * p.tiles);
    // (a tree's parts are larger, for its rows, and so is the work of each step: 64 sequences of 8 key heads of up to 2048
    // slots, 32 rows, 51 us with four parts, 31 with one; 16 of 4096, 40 rows, 35 with eight, 33)
    if (tree && few) want = bh * p.tiles >= cus ? 1 : (2 * (int64_t)cus + bh * p.tiles - 1) / (bh * p.tiles);
    const int64_t able = (most + 4 * step - 1) / (4 * step);
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, able), 256));
    // (computing the scores again instead, one token of 16 x 8 x 8192 slots at most, D = 128: 4
    // rows 28 and 97 us, 32 rows 73 and 121; the workspace that they take is kept below 4 GiB)
    p.scores = a->accumulate && rows <= 32 && (uint64_t)bh * rows * most < (uint64_t(1) << 30);
    uint64_t at = 0;
    auto take = [&](uint64_t n) {
        const uint64_t here = at;
        at += (n + 255) / 256 * 256;
        return here;
    };
    if (p.splits > 1) p.part_o = take((uint64_t)p.splits * bh * rows * a->cache.head_dim * 4);
    if (p.splits > 1 || p.scores) p.part_ml = take((uint64_t)p.splits * bh * rows * 8);
    if (a->accumulate && !p.scores) p.row_lse = take((uint64_t)bh * rows * 4);
    if (p.scores) p.scores_at = take((uint64_t)bh * rows * most * 4);
    const int wg_keys = p.scores ? 1024 : a->cache.head_dim == 256 ? Weigh<256>::WG_KEYS : Weigh<128>::WG_KEYS;
    p.weight_tiles = (int)((most + wg_keys - 1) / wg_keys);
    p.weight_parts = 1;
    if (a->accumulate && !p.scores) {
        const int64_t fill = (2 * (int64_t)cus + bh * p.weight_tiles - 1) / (bh * p.weight_tiles);
        p.weight_parts = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(fill, rows / 128), 64));
        if (p.weight_parts > 1) p.part_w = take((uint64_t)p.weight_parts * bh * most * 4);
    }
    p.bytes = at;
    return p;
}

int cus_of_current_device() {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1)
        return 256;
    return n;
}

template <class T, int D, int MASK>
const void* attend_fn(const Plan& p) {
    if (p.few) {
        if constexpr (D <= 128)
            if (p.nb == 2) return (const void*)&attend_kernel<T, D, 2, MASK>;
        return (const void*)&attend_kernel<T, D, 1, MASK>;
    }
    if constexpr (MASK == MASK_TREE && D <= 128)
        if (p.groups == 2) return (const void*)&attend_many_kernel<T, D, MASK, 8, 2>;
    if constexpr (D == 256)
        if (p.waves == 4) return (const void*)&attend_many_kernel<T, D, MASK, 4>;
    return (const void*)&attend_many_kernel<T, D, MASK, 8>;
}

struct Functions {
    const void *attend, *finish, *weights;
};

template <class T, int D>
Functions functions(const Plan& p, int mask) {
    return {mask == MASK_TREE       ? attend_fn<T, D, MASK_TREE>(p)
            : mask == MASK_POSITION ? attend_fn<T, D, MASK_POSITION>(p)
                                    : attend_fn<T, D, MASK_NONE>(p),
            (const void*)&finish_kernel<T, D>,
            mask == MASK_POSITION ? (const void*)&weights_kernel<T, D, true> : (const void*)&weights_kernel<T, D, false>};
}

template <class T>
Functions functions(const Plan& p, int mask, int64_t d) {
    switch (d) {
        case 32: return functions<T, 32>(p, mask);
        case 64: return functions<T, 64>(p, mask);
        case 128: return functions<T, 128>(p, mask);
        default: return functions<T, 256>(p, mask);
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

int attend(const rsfa_cache4_attend_args* a, const int32_t* tree, int64_t tree_stride, int mask, void* stream) {
    int st = check_attend(a);
    if (st != RSFA_OK) return st;
    if (!a->q || !a->o) return RSFA_E_NULL;
    if ((st = check_rows(a->q, a->q_stride)) != RSFA_OK || (st = check_rows(a->o, a->o_stride)) != RSFA_OK) return st;
    if (((uintptr_t)a->lse | (uintptr_t)a->lengths | (uintptr_t)a->counts | (uintptr_t)a->pos_start) & 3)
        return RSFA_E_ALIGN;
    const Plan plan = make_plan(a, cus_of_current_device(), mask == MASK_TREE);
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
    // (a scale of 0 would make a hidden score -inf * 0; at FLT_MIN the others still have weights of 1)
    p.scale = std::max(__builtin_fabsf(a->sm_scale) * LOG2E, FLT_MIN);
    p.neg = a->sm_scale < 0.0f ? 0x80008000u : 0u;
    char* ws = (char*)a->workspace;
    if (plan.splits > 1) p.part_o = (float*)(ws + plan.part_o);
    if (plan.splits > 1 || plan.scores) p.part_ml = (float2*)(ws + plan.part_ml);
    if (a->accumulate && !plan.scores) p.row_lse = (float*)(ws + plan.row_lse);
    if (plan.scores) p.scores = (float*)(ws + plan.scores_at);
    p.tree = (const uint32_t*)tree;
    p.tree_sz = tree_stride;
    p.tree_words = (p.t + 31) / 32;
    const Functions fn = a->cache.dtype == RSFA_DTYPE_BF16 ? functions<BF16>(plan, mask, a->cache.head_dim)
                                                           : functions<F16>(plan, mask, a->cache.head_dim);
    const int64_t grid = (int64_t)p.bh * plan.tiles;
    const int64_t weight_grid = (int64_t)p.bh * plan.weight_tiles;
    const int64_t join_grid = (int64_t)p.bh * ((p.most + 255) / 256);
    if (grid > 0x7fffffff || (a->accumulate && join_grid > 0x7fffffff)) return RSFA_E_CACHE;
    void* args[] = {&p};
    if (hipLaunchKernel(fn.attend, dim3((unsigned)grid, (unsigned)plan.splits), dim3(64 * plan.waves), args, 0, (hipStream_t)stream) != hipSuccess)
        return RSFA_E_LAUNCH;
    if (plan.splits > 1 || plan.scores) {
        const int64_t rows = (int64_t)p.bh * p.rows;
        const int groups = 256 / (int)(a->cache.head_dim / 4);
        int pp = 1;
        while (pp < groups && pp * 8 < plan.splits) pp *= 2;
        const int64_t per = groups / pp;
        int join_blocks = plan.splits > 1 ? (int)((rows + per - 1) / per) : 0;
        const int64_t blocks = join_blocks + (plan.scores ? weight_grid : 0);
        if (blocks > 0x7fffffff) return RSFA_E_CACHE;
        void* finish_args[] = {&p, &pp, &join_blocks};
        if (hipLaunchKernel(fn.finish, dim3((unsigned)blocks), dim3(256), finish_args, 0, (hipStream_t)stream) != hipSuccess)
            return RSFA_E_LAUNCH;
    }
    if (a->accumulate && !plan.scores) {
        if (plan.weight_parts > 1) p.part_w = (float*)(ws + plan.part_w);
        const int threads = 64 * (a->cache.head_dim == 256 ? Weigh<256>::WAVES : Weigh<128>::WAVES);
        if (hipLaunchKernel(fn.weights, dim3((unsigned)weight_grid, (unsigned)plan.weight_parts), dim3(threads), args, 0, (hipStream_t)stream) != hipSuccess)
            return RSFA_E_LAUNCH;
        if (plan.weight_parts > 1) {
            int parts = plan.weight_parts;
            void* join_args[] = {&p, &parts};
            if (hipLaunchKernel((const void*)&join_weights_kernel, dim3((unsigned)join_grid), dim3(256), join_args, 0, (hipStream_t)stream) != hipSuccess)
                return RSFA_E_LAUNCH;
        }
    }
    return RSFA_OK;
}

}  // namespace

extern "C" {

uint64_t rsfa_cache4_attend_workspace_bytes(const rsfa_cache4_attend_args* a) {
    if (check_attend(a) != RSFA_OK) return 0;
    return make_plan(a, cus_of_current_device(), false).bytes;
}

uint64_t rsfa_cache4_attend_tree_workspace_bytes(const rsfa_cache4_attend_args* a) {
    if (check_attend(a) != RSFA_OK) return 0;
    return make_plan(a, cus_of_current_device(), true).bytes;
}

int rsfa_cache4_attend(const rsfa_cache4_attend_args* a, void* stream) {
    return attend(a, nullptr, 0, a && a->causal ? MASK_POSITION : MASK_NONE, stream);
}

int rsfa_cache4_attend_tree(const rsfa_cache4_attend_args* a, const int32_t* bits, int64_t bits_stride, void* stream) {
    if (!a || !bits) return RSFA_E_NULL;
    if (a->struct_size != sizeof(rsfa_cache4_attend_args)) return RSFA_E_ABI;
    if ((uintptr_t)bits & 3) return RSFA_E_ALIGN;
    if (a->accumulate || a->pos_start || a->t > RSFA_DRAFT_TOKENS || bits_stride < 0) return RSFA_E_DRAFT;
    return attend(a, bits, bits_stride, MASK_TREE, stream);
}

}  // extern "C"
