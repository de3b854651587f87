// Rows of a 4-bit cache: append (quantise and write) and read (their values).
//
// Four lanes share a block of 32 values, eight values (one 16-byte load, one
// dword of codes) each, so a wave's accesses are whole rows; the block's largest
// magnitude takes two exchanges between neighbouring lanes.  Scaling by a power of
// two is exact, and v_cvt_scalef32_pk_fp4_f32 rounds x / 2^e to the nearest
// code, ties to even, magnitudes above 6 to 6 (checked for every float16 value).
// Both are bound by memory: 2 D bytes a row on one side, D/2 + D/32 on the other.
//
// Of tokens that name one slot the last has it.  With few tokens each looks through
// those after it.  With many that would be quadratic in them, so the slots themselves say whose they are, in what the
// call overwrites: the first word of a slot's K codes takes the largest token + 1 that names
// it (cleared, then atomic maxima, whose order has no say); its owner writes V and the
// position, which no other token of the sequence has; then K goes by the position.
#include "cache4.hpp"

using namespace rsfa4;

namespace {

struct RowsParams {
    rsfa_cache4 c;
    const char* src[2];  // append: k, v
    char* dst[2];        // read: k, v
    int64_t st[2][3];    // their element strides of (Z, H, T)
    const int32_t *lengths, *slots, *counts, *pos_start;
    int64_t length;
    uint32_t t, h, rows;  // rows = Z * H * T
    uint32_t blocks;      // append, several rows a thread: blocks of a head's tokens
    int32_t owners;       // how append with slots finds a slot's owner: LOOK, or in two launches BY_TOKEN (V), BY_POSITION (K)
};

constexpr int LOOK = 0, BY_TOKEN = 1, BY_POSITION = 2;

struct Row {
    int z, h;
    uint32_t t;
};

__device__ __forceinline__ Row row_of(const RowsParams& p, uint32_t r) {
    Row o;
    const uint32_t zh = r / p.t;
    o.t = r - zh * p.t;
    o.z = (int)(zh / p.h);
    o.h = (int)(zh - o.z * p.h);
    return o;
}

__device__ __forceinline__ int64_t code_at(const rsfa_cache4& c, const Row& w, int64_t slot, int d) {
    return w.z * c.code_stride[0] + w.h * c.code_stride[1] + slot * (d / 2);
}
__device__ __forceinline__ int64_t scale_at(const rsfa_cache4& c, const Row& w, int64_t slot, int d) {
    return w.z * c.scale_stride[0] + w.h * c.scale_stride[1] + slot * (d / 32);
}
__device__ __forceinline__ int64_t slot_at(const rsfa_cache4& c, const Row& w, int64_t slot) {
    return w.z * c.slot_stride[0] + w.h * c.slot_stride[1] + slot;
}

__device__ __forceinline__ uint32_t* owner_of(const RowsParams& p, const Row& w, int64_t slot) {
    return (uint32_t*)(p.c.k_codes + code_at(p.c, w, slot, (int)p.c.head_dim));
}

// Position of a row's token.
__device__ __forceinline__ int32_t position_of(const RowsParams& p, const Row& w) {
    const int64_t start = p.pos_start ? (int64_t)p.pos_start[w.z] : length_of(p.lengths, p.length, w.z, p.c.capacity);
    return (int32_t)(start + w.t);
}

// The slot that a row's token names, or -1: past the sequence's count or outside the cache.
__device__ __forceinline__ int64_t named(const RowsParams& p, const Row& w, uint32_t r) {
    if (p.counts && (int64_t)w.t >= p.counts[w.z]) return -1;
    const int64_t s = p.slots ? (int64_t)p.slots[r] : length_of(p.lengths, p.length, w.z, p.c.capacity) + (int64_t)w.t;
    return s >= 0 && s < p.c.capacity ? s : -1;
}

// The slot that a row's token has, or -1: none, or one that a later token has.
__device__ __forceinline__ int64_t target(const RowsParams& p, const Row& w, uint32_t r) {
    const int64_t s = named(p, w, r);
    if (s < 0 || !p.slots) return s;
    if (p.owners == BY_TOKEN) return *owner_of(p, w, s) == w.t + 1 ? s : -1;
    if (p.owners == BY_POSITION) return p.c.positions[slot_at(p.c, w, s)] == position_of(p, w) ? s : -1;
    const int64_t end = p.counts && p.counts[w.z] < (int64_t)p.t ? p.counts[w.z] : (int64_t)p.t;
    for (int64_t i = w.t + 1; i < end; ++i)
        if (p.slots[r + (i - w.t)] == s) return -1;
    return s;
}

// Owners of the slots: cleared, then the largest token + 1 that names each.
template <bool CLEAR>
__global__ void __launch_bounds__(256) owners_kernel(RowsParams p) {
    const uint32_t r = blockIdx.x * 256 + threadIdx.x;
    if (r >= p.rows) return;
    const Row w = row_of(p, r);
    const int64_t s = named(p, w, r);
    if (s < 0) return;
    if (CLEAR) *owner_of(p, w, s) = 0;
    else atomicMax(owner_of(p, w, s), w.t + 1);
}

// One thread: eight values of EACH K (blockIdx.y = 0) or V rows, PER_BLOCK rows apart.
// Four rows' loads are under way together where there are rows for it (4 x 3977 tokens
// of 8 heads, D = 128, bf16: append 24.2 -> 22.6 us, read 18.9 -> 16.9; floors at the
// rate of a large copy 15.9 each); one row each where there are few (512 rows: append 4.3,
// with four 6.3).
template <class T, int D, int EACH>
__global__ void __launch_bounds__(256) append_kernel(RowsParams p) {
    constexpr int LANES = D / 8, PER_BLOCK = 256 / LANES;
    typedef typename T::x8 x8;
    const int lane = threadIdx.x % LANES;
    const int v = p.owners == LOOK ? (int)blockIdx.y : p.owners == BY_TOKEN;
    Row w[EACH];
    uint32_t rows[EACH];
    x8 in[EACH];
    if constexpr (EACH > 1) {
        // a block of tokens of one head; the heads of the same tokens are neighbours in the
        // grid, as [Z, T, H, D] tensors have them in memory
        const uint32_t rest = blockIdx.x / p.h;
        const uint32_t z = rest / p.blocks, h = blockIdx.x - rest * p.h;
        const uint32_t t0 = (rest - z * p.blocks) * (PER_BLOCK * EACH) + threadIdx.x / LANES;
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            w[e].z = (int)z, w[e].h = (int)h, w[e].t = t0 + e * PER_BLOCK;
            rows[e] = w[e].t < p.t ? (z * p.h + h) * p.t + w[e].t : p.rows;
        }
    } else {
        rows[0] = blockIdx.x * PER_BLOCK + threadIdx.x / LANES;
        w[0] = row_of(p, min(rows[0], p.rows - 1));
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e)
        in[e] = *(const x8*)((const typename T::elem*)p.src[v] + w[e].z * p.st[v][0] + w[e].h * p.st[v][1] +
                             min(w[e].t, p.t - 1) * p.st[v][2] + 8 * lane);
    uint8_t* cb = v ? p.c.v_codes : p.c.k_codes;
    uint8_t* sb = v ? p.c.v_scales : p.c.k_scales;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        if (rows[e] >= p.rows) return;  // whole blocks of four lanes leave together
        const int64_t slot = target(p, w[e], rows[e]);
        if (slot < 0) continue;
        float x[8];
        // (bits order as magnitudes do, infinities and NaN above all others)
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = (float)in[e][i];
            top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
        }
        top = max(top, (uint32_t)__shfl_xor((int)top, 1));
        top = max(top, (uint32_t)__shfl_xor((int)top, 2));
        // 7 * 2^e = 1.75 * 2^(e + 2): the exponent less 2, one more past 1.75
        int ex = (int)(top >> 23) - 127 - 2 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
        ex = ex < T::lo ? T::lo : ex > T::hi ? T::hi : ex;
        const bool nan = top >= 0x7f800000u;
        const uint32_t byte = nan ? 255u : (uint32_t)(ex + 127);
        const float scale = __uint_as_float((uint32_t)(ex + 127) << 23);
        uint32_t codes = 0;
        if (!nan) {
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], scale, 0);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
        }
        *(uint32_t*)(cb + code_at(p.c, w[e], slot, D) + 4 * lane) = codes;
        if ((lane & 3) == 0) sb[scale_at(p.c, w[e], slot, D) + lane / 4] = (uint8_t)byte;
        if ((v == 0) == (p.owners == LOOK) && lane == 0) {
            const int64_t at = slot_at(p.c, w[e], slot);
            p.c.positions[at] = position_of(p, w[e]);
            if (p.c.weights) p.c.weights[at] = 0.0f;
        }
    }
}

template <class T, int D, int EACH>
__global__ void __launch_bounds__(256) read_kernel(RowsParams p) {
    constexpr int LANES = D / 8, PER_BLOCK = 256 / LANES;
    const int v = blockIdx.y;
    if (!p.dst[v]) return;
    const int lane = threadIdx.x % LANES;
    const uint32_t first = blockIdx.x * (PER_BLOCK * EACH) + threadIdx.x / LANES;
    const uint8_t* cb = v ? p.c.v_codes : p.c.k_codes;
    const uint8_t* sb = v ? p.c.v_scales : p.c.k_scales;
    Row w[EACH];
    uint32_t codes[EACH], scale[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const uint32_t r = min(first + e * PER_BLOCK, p.rows - 1);
        w[e] = row_of(p, r);
        const int64_t slot = p.slots ? (int64_t)p.slots[r] : (p.lengths ? (int64_t)p.lengths[w[e].z] : p.length) + w[e].t;
        codes[e] = scale[e] = 0;
        if (slot >= 0 && slot < p.c.capacity) {
            codes[e] = *(const uint32_t*)(cb + code_at(p.c, w[e], slot, D) + 4 * lane);
            scale[e] = sb[scale_at(p.c, w[e], slot, D) + lane / 4];
        }
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        if (first + e * PER_BLOCK >= p.rows) return;
        const float s = __uint_as_float(scale[e] << 23);
        u32x4 out;  // (codes and scale of 0 are zeros)
        out[0] = T::template cvt<0>(codes[e], s);
        out[1] = T::template cvt<1>(codes[e], s);
        out[2] = T::template cvt<2>(codes[e], s);
        out[3] = T::template cvt<3>(codes[e], s);
        *(u32x4*)((typename T::elem*)p.dst[v] + w[e].z * p.st[v][0] + w[e].h * p.st[v][1] + w[e].t * p.st[v][2] + 8 * lane) = out;
    }
}

// Tokens that look through those after them: T = 64, 96, 128, 1024 tokens of 4 sequences and 8 heads, D = 128, take 9.5,
// 13, 16, 277 us so, and 10.2, 10.5, 10.7, 17 by owners (in a graph; a call of four launches of its
// own 17 where one takes 10, 14, 17); 4096 tokens 4600 and 45, where consecutive slots take 19.
constexpr int64_t LOOKED = 96;

template <class T, int EACH>
const void* pick(bool read, int64_t d) {
    switch (d) {
        case 32: return read ? (const void*)&read_kernel<T, 32, EACH> : (const void*)&append_kernel<T, 32, EACH>;
        case 64: return read ? (const void*)&read_kernel<T, 64, EACH> : (const void*)&append_kernel<T, 64, EACH>;
        case 128: return read ? (const void*)&read_kernel<T, 128, EACH> : (const void*)&append_kernel<T, 128, EACH>;
        default: return read ? (const void*)&read_kernel<T, 256, EACH> : (const void*)&append_kernel<T, 256, EACH>;
    }
}

int rows_launch(const rsfa_cache4_rows_args* a, bool read, void* stream) {
    if (!a) return RSFA_E_NULL;
    if (a->struct_size != sizeof(rsfa_cache4_rows_args)) return RSFA_E_ABI;
    int st = check_cache(a->cache, false);
    if (st != RSFA_OK) return st;
    if (read ? !a->k && !a->v : !a->k || !a->v) return RSFA_E_NULL;
    if (a->t < 1 || a->t > (1 << 30)) return RSFA_E_CACHE;
    if (a->k && (st = check_rows(a->k, a->k_stride)) != RSFA_OK) return st;
    if (a->v && (st = check_rows(a->v, a->v_stride)) != RSFA_OK) return st;
    if (((uintptr_t)a->lengths | (uintptr_t)a->slots | (uintptr_t)a->counts | (uintptr_t)a->pos_start) & 3)
        return RSFA_E_ALIGN;
    RowsParams p{};
    p.c = a->cache;
    p.src[0] = (const char*)a->k, p.src[1] = (const char*)a->v;
    p.dst[0] = (char*)a->k, p.dst[1] = (char*)a->v;
    for (int i = 0; i < 3; ++i) p.st[0][i] = a->k_stride[i], p.st[1][i] = a->v_stride[i];
    p.lengths = a->lengths, p.slots = a->slots, p.length = a->length;
    p.counts = read ? nullptr : a->counts, p.pos_start = read ? nullptr : a->pos_start;
    const int64_t rows = a->cache.z * a->cache.h * a->t;
    if (rows > 0x7fffffff) return RSFA_E_CACHE;
    p.t = (uint32_t)a->t, p.h = (uint32_t)a->cache.h, p.rows = (uint32_t)rows;
    // four rows a thread once one each would be over eight workgroups on each of 256 CUs
    const int64_t one = 256 / (a->cache.head_dim / 8);
    // (append: where a head's tokens fill a block of four rows a thread)
    const bool four = rows > 2048 * one && (read || a->t >= 4 * one);
    const int64_t per = four ? 4 * one : one;
    int64_t blocks = (rows + per - 1) / per;
    if (four && !read) {
        p.blocks = (uint32_t)((a->t + per - 1) / per);
        blocks = a->cache.z * a->cache.h * p.blocks;
    }
    const int64_t d = a->cache.head_dim;
    const void* fn = a->cache.dtype == RSFA_DTYPE_BF16 ? (four ? pick<BF16, 4>(read, d) : pick<BF16, 1>(read, d))
                                                       : (four ? pick<F16, 4>(read, d) : pick<F16, 1>(read, d));
    void* args[] = {&p};
    auto launch = [&](const void* f, dim3 grid) {
        return hipLaunchKernel(f, grid, dim3(256), args, 0, (hipStream_t)stream) == hipSuccess;
    };
    if (read || !a->slots || a->t <= LOOKED) return launch(fn, dim3((unsigned)blocks, 2)) ? RSFA_OK : RSFA_E_LAUNCH;
    const dim3 all((unsigned)((rows + 255) / 256));
    if (!launch((const void*)&owners_kernel<true>, all) || !launch((const void*)&owners_kernel<false>, all)) return RSFA_E_LAUNCH;
    p.owners = BY_TOKEN;
    if (!launch(fn, dim3((unsigned)blocks))) return RSFA_E_LAUNCH;
    p.owners = BY_POSITION;
    return launch(fn, dim3((unsigned)blocks)) ? RSFA_OK : RSFA_E_LAUNCH;
}

}  // namespace

extern "C" {

int rsfa_cache4_append(const rsfa_cache4_rows_args* a, void* stream) { return rows_launch(a, false, stream); }
int rsfa_cache4_read(const rsfa_cache4_rows_args* a, void* stream) { return rows_launch(a, true, stream); }

}  // extern "C"
