// Rotary positions (rsfa_rotary, declared in include/rsfa.h).
//
// Pair i of a head of the token at position p is turned by the angle
// a = 2 pi p turns[i]: (u, w) -> amplitude * (u cos a - w sin a, w cos a + u sin a).
//
// What bounds it: memory; every value is read and written once.  The angles come from the positions and the
// R/2 frequencies in the kernel, so no table of cosines is read; a thread
// turns the same pairs of a few heads, so an angle is computed once for
// them.  The reduction of p * turns[i] to a fraction of a
// turn is in 64 bits (at p = 2^20 a 32-bit product is off by 2^-4 turns); the
// sine and cosine of the fraction, the products and sums are in 32 bits, and each
// output is rounded to its type once.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "../../include/rsfa.h"

namespace {

struct RotaryParams {
    const char* x[2];
    char* y[2];
    int64_t xs[2][3], ys[2][3];  // element strides of (Z, H, N)
    int32_t heads[2];
    const void* positions;
    int64_t ps[2], start;
    const double* turns;
    float amplitude;
    int32_t pos64, inverse;
    int64_t n, tokens;      // tokens = Z * N
    int32_t half;           // R / 2
    int32_t rotary, dim;    // R, D
    int32_t pair_units, copy_units;  // threads of a token that turn pairs / copy the rest of the head
    int32_t hpt;            // heads per thread
    uint32_t groups;        // of hpt heads
};

template <class E, int V>
struct alignas(sizeof(E) * V) Vec {
    E v[V];
};

// Sine and cosine of 2 pi p f, scaled.  The fraction of a turn goes into them in 32 bits (2^-26 of a turn, 1.6 * 2^-24
// radians at most): of the three types only float32 has steps as small, and 64-bit sines would take many
// times the instructions.
__device__ __forceinline__ void angle(double p, double f, float amp, bool inverse, float& s, float& c) {
    const double turn = p * f;
    float frac = (float)(turn - __builtin_rint(turn));
    if (inverse) frac = -frac;
    sincospif(2.0f * frac, &s, &c);
    s *= amp;
    c *= amp;
}

// A unit of a token is V pairs, or 2 V values that are copied: one thread's work on
// each of its heads, two loads and two stores of V elements.  Its two chunks lie R/2
// apart (half the copied values apart) in either layout, so that neighbouring lanes
// load neighbouring chunks; interleaved pairs with V > 1 lie inside a chunk.
template <class E, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryParams p) {
    typedef Vec<E, V> Chunk;
    constexpr bool INSIDE = INTERLEAVED && V > 1;
    const int units = p.pair_units + p.copy_units;
    const uint32_t block = blockIdx.x / p.groups, hg = blockIdx.x - block * p.groups;
    const int64_t id = (int64_t)block * 256 + threadIdx.x;
    const int64_t token = id / units;
    if (token >= p.tokens) return;
    const int u = (int)(id - token * units);
    const int64_t z = token / p.n, n = token - z * p.n;
    const bool turns = u < p.pair_units;
    int a, b;  // the first values of the unit's two chunks
    bool two = true;
    float c[V], s[V];
    if (turns) {
        a = INTERLEAVED && V == 1 ? 2 * u : V * u;
        b = INTERLEAVED && V == 1 ? a + 1 : a + p.half;
        int64_t pos = p.start + n;
        if (p.positions) {
            const int64_t at = z * p.ps[0] + n * p.ps[1];
            pos = p.pos64 ? ((const int64_t*)p.positions)[at] : (int64_t)((const int32_t*)p.positions)[at];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int pair = INSIDE ? (i < V / 2 ? a / 2 + i : b / 2 + i - V / 2) : V * u + i;
            angle((double)pos, p.turns[pair], p.amplitude, p.inverse != 0, s[i], c[i]);
        }
    } else {
        a = p.rotary + V * (u - p.pair_units);
        b = a + V * p.copy_units;
        two = b < p.dim;
    }
    const int first = (int)hg * p.hpt;
    const int last = min(first + p.hpt, p.heads[0] + p.heads[1]);
#pragma unroll 4
    for (int h = first; h < last; ++h) {
        const int t = h >= p.heads[0];
        const int64_t lh = t ? h - p.heads[0] : h;
        const E* x = (const E*)p.x[t] + z * p.xs[t][0] + lh * p.xs[t][1] + n * p.xs[t][2];
        E* y = (E*)p.y[t] + z * p.ys[t][0] + lh * p.ys[t][1] + n * p.ys[t][2];
        Chunk lo = *(const Chunk*)(x + a), hi = lo;
        if (two) hi = *(const Chunk*)(x + b);
        if (turns) {
            auto turn = [](E& eu, E& ew, float cos, float sin) {
                const float fu = (float)eu, fw = (float)ew;
                eu = (E)(fu * cos - fw * sin);
                ew = (E)(fw * cos + fu * sin);
            };
            if constexpr (INSIDE) {
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    turn(lo.v[2 * i], lo.v[2 * i + 1], c[i], s[i]);
                    turn(hi.v[2 * i], hi.v[2 * i + 1], c[V / 2 + i], s[V / 2 + i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) turn(lo.v[i], hi.v[i], c[i], s[i]);
            }
        }
        *(Chunk*)(y + a) = lo;
        if (two) *(Chunk*)(y + b) = hi;
    }
}

template <class E, int V>
const void* pick(bool interleaved) {
    return interleaved ? (const void*)&rotary_kernel<E, V, true> : (const void*)&rotary_kernel<E, V, false>;
}

}  // namespace

extern "C" int rsfa_rotary(const rsfa_rotary_args* a, void* stream) {
    if (!a) return RSFA_E_NULL;
    if (a->struct_size != sizeof(rsfa_rotary_args)) return RSFA_E_ABI;
    if (!a->x[0] || !a->y[0] || (!a->x[1] != !a->y[1]) || !a->turns) return RSFA_E_NULL;
    if (a->dtype != RSFA_DTYPE_F16 && a->dtype != RSFA_DTYPE_BF16 && a->dtype != RSFA_DTYPE_F32) return RSFA_E_DTYPE;
    const int tensors = a->x[1] ? 2 : 1;
    if (a->z < 1 || a->n < 1 || a->z > (1 << 30) || a->n > (1 << 30) || a->z * a->n > (int64_t(1) << 40))
        return RSFA_E_SHAPE;
    if (a->head_dim < 2 || a->head_dim > 65536 || a->rotary_dim < 2 || a->rotary_dim > a->head_dim ||
        (a->rotary_dim & 1))
        return RSFA_E_ROTARY;
    const int size = a->dtype == RSFA_DTYPE_F32 ? 4 : 2;
    const int wide = 16 / size;
    // wide loads need 16-byte rows and pairs that fill them
    bool aligned = a->rotary_dim % (2 * wide) == 0 && a->head_dim % wide == 0;
    int64_t all = 0;
    for (int i = 0; i < tensors; ++i) {
        if (a->heads[i] < 1 || a->heads[i] > (1 << 20)) return RSFA_E_SHAPE;
        all += a->heads[i];
        if (a->x_stride[i][3] != 1 || a->y_stride[i][3] != 1) return RSFA_E_ALIGN;
        if (((uintptr_t)a->x[i] | (uintptr_t)a->y[i]) & (size - 1)) return RSFA_E_ALIGN;
        for (int d = 0; d < 3; ++d)
            if (a->x[i] == a->y[i] && a->x_stride[i][d] != a->y_stride[i][d]) return RSFA_E_ALIGN;
        aligned = aligned && !(((uintptr_t)a->x[i] | (uintptr_t)a->y[i]) & 15);
        for (int d = 0; d < 3; ++d) aligned = aligned && a->x_stride[i][d] % wide == 0 && a->y_stride[i][d] % wide == 0;
    }
    if ((uintptr_t)a->turns & 7) return RSFA_E_ALIGN;
    if ((uintptr_t)a->positions & (a->flags & RSFA_ROTARY_POS64 ? 7 : 3)) return RSFA_E_ALIGN;
    RotaryParams p{};
    for (int i = 0; i < tensors; ++i) {
        p.x[i] = (const char*)a->x[i];
        p.y[i] = (char*)a->y[i];
        for (int d = 0; d < 3; ++d) p.xs[i][d] = a->x_stride[i][d], p.ys[i][d] = a->y_stride[i][d];
        p.heads[i] = (int32_t)a->heads[i];
    }
    p.positions = a->positions;
    p.ps[0] = a->pos_stride[0], p.ps[1] = a->pos_stride[1];
    p.start = a->start;
    p.turns = a->turns;
    p.amplitude = a->amplitude;
    p.pos64 = a->flags & RSFA_ROTARY_POS64 ? 1 : 0;
    p.inverse = a->flags & RSFA_ROTARY_INVERSE ? 1 : 0;
    p.n = a->n;
    p.tokens = a->z * a->n;
    p.half = (int32_t)(a->rotary_dim / 2);
    p.rotary = (int32_t)a->rotary_dim;
    p.dim = (int32_t)a->head_dim;
    const int V = aligned ? wide : 1;
    p.pair_units = p.half / V;
    p.copy_units = (int32_t)((a->head_dim - a->rotary_dim + 2 * V - 1) / (2 * V));
    // values that are not turned stay where they are when the call is in place
    bool in_place = true;
    for (int i = 0; i < tensors; ++i) in_place = in_place && a->x[i] == a->y[i];
    if (in_place) p.copy_units = 0;
    const int64_t threads = p.tokens * (p.pair_units + p.copy_units);
    const int64_t blocks = (threads + 255) / 256;
    if (blocks > 0x7fffffff) return RSFA_E_SHAPE;
    // Heads that a thread takes one after another, with the same angles: few, so that
    // the workgroups of a token's heads, which are neighbours in the grid, pass over memory
    // side by side (8 x 4093 tokens of 32 heads, bf16, [Z, N, H, D], forward and backward,
    // with 2, 4, 8, 16, 32 heads: 222, 224, 230, 270, 287 us; 4096 tokens in [Z, H, N, D]
    // forward 94, 99, 103; float32, 4 x 2048 tokens of 20 heads 19.8, 14.5, 15.1); without
    // wide loads, where the angles cost more, eight (2, 4, 8: 45, 38, 34).
    int64_t hpt = std::min<int64_t>(all, V > 1 ? 4 : 8);
    while (hpt > 1 && blocks * ((all + hpt - 1) / hpt) < 2048) hpt = (hpt + 1) / 2;
    p.hpt = (int32_t)hpt;
    p.groups = (uint32_t)((all + hpt - 1) / hpt);
    const int64_t grid = blocks * p.groups;
    if (grid > 0x7fffffff) return RSFA_E_SHAPE;
    const bool il = a->flags & RSFA_ROTARY_INTERLEAVED;
    const void* fn = a->dtype == RSFA_DTYPE_F32    ? (V > 1 ? pick<float, 4>(il) : pick<float, 1>(il))
                     : a->dtype == RSFA_DTYPE_BF16 ? (V > 1 ? pick<__bf16, 8>(il) : pick<__bf16, 1>(il))
                                                   : (V > 1 ? pick<_Float16, 8>(il) : pick<_Float16, 1>(il));
    void* args[] = {&p};
    if (hipLaunchKernel(fn, dim3((unsigned)grid), dim3(256), args, 0,
                        (hipStream_t)stream) != hipSuccess)
        return RSFA_E_LAUNCH;
    return RSFA_OK;
}
