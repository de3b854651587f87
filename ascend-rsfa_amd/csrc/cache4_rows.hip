// Rows of a 4-bit cache: append (quantise and write) and read (their values).
//
// Four lanes share a block of 32 values, eight values (one 16-byte load, one
// dword of codes) each, so a wave's accesses are whole rows; the block's largest
// magnitude takes two exchanges between neighbouring lanes.  Scaling by a power of
// two is exact, and v_cvt_scalef32_pk_fp4_f32 rounds x / 2^e to the nearest
// code, ties to even, magnitudes above 6 to 6 (checked for every float16 value).
// Both are bound by memory: 2 D bytes a row on one side, D/2 + D/32 on the other.
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
    int64_t t, rows;     // rows = Z * H * T
};

struct Row {
    int z, h;
    int64_t t;
};

__device__ __forceinline__ Row row_of(const RowsParams& p, int64_t r) {
    Row o;
    const int64_t zh = r / p.t;
    o.t = r - zh * p.t;
    o.z = (int)(zh / p.c.h);
    o.h = (int)(zh - (int64_t)o.z * p.c.h);
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

// The slot of a row's token, or -1: past the sequence's count, outside the
// cache, or named again by a later token.
__device__ __forceinline__ int64_t target(const RowsParams& p, const Row& w, int64_t r) {
    if (p.counts && w.t >= p.counts[w.z]) return -1;
    int64_t s;
    if (p.slots) {
        s = p.slots[r];
        const int64_t end = p.counts && p.counts[w.z] < p.t ? p.counts[w.z] : p.t;
        for (int64_t i = w.t + 1; i < end; ++i)
            if (p.slots[r + (i - w.t)] == s) return -1;
    } else {
        s = length_of(p.lengths, p.length, w.z, p.c.capacity) + w.t;
    }
    return s >= 0 && s < p.c.capacity ? s : -1;
}

// One thread: eight values of a K (blockIdx.y = 0) or V row.
template <class T, int D>
__global__ void __launch_bounds__(256) append_kernel(RowsParams p) {
    constexpr int LANES = D / 8;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t r = id / LANES;
    if (r >= p.rows) return;  // whole blocks of four lanes leave together
    const int lane = (int)(id - r * LANES);
    const Row w = row_of(p, r);
    const int64_t slot = target(p, w, r);
    if (slot < 0) return;
    const int v = blockIdx.y;
    typedef typename T::x8 x8;
    const typename T::elem* src = (const typename T::elem*)p.src[v] + w.z * p.st[v][0] + w.h * p.st[v][1] + w.t * p.st[v][2];
    const x8 in = *(const x8*)(src + 8 * lane);
    float x[8];
    // (bits order as magnitudes do, infinities and NaN above all others)
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = (float)in[i];
        top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    // 7 * 2^e = 1.75 * 2^(e + 2): e is the exponent less 2, one more past 1.75
    int e = (int)(top >> 23) - 127 - 2 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = e < T::lo ? T::lo : e > T::hi ? T::hi : e;
    const bool nan = top >= 0x7f800000u;
    const uint32_t byte = nan ? 255u : (uint32_t)(e + 127);
    const float scale = __uint_as_float((uint32_t)(e + 127) << 23);
    uint32_t codes = 0;
    if (!nan) {
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], scale, 0);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], scale, 1);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], scale, 2);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], scale, 3);
    }
    uint8_t* cb = v ? p.c.v_codes : p.c.k_codes;
    uint8_t* sb = v ? p.c.v_scales : p.c.k_scales;
    *(uint32_t*)(cb + code_at(p.c, w, slot, D) + 4 * lane) = codes;
    if ((lane & 3) == 0) sb[scale_at(p.c, w, slot, D) + lane / 4] = (uint8_t)byte;
    if (v == 0 && lane == 0) {
        const int64_t at = slot_at(p.c, w, slot);
        const int64_t first = p.pos_start ? (int64_t)p.pos_start[w.z] : length_of(p.lengths, p.length, w.z, p.c.capacity);
        p.c.positions[at] = (int32_t)(first + w.t);
        if (p.c.weights) p.c.weights[at] = 0.0f;
    }
}

template <class T, int D>
__global__ void __launch_bounds__(256) read_kernel(RowsParams p) {
    constexpr int LANES = D / 8;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t r = id / LANES;
    if (r >= p.rows) return;
    const int v = blockIdx.y;
    if (!p.dst[v]) return;
    const int lane = (int)(id - r * LANES);
    const Row w = row_of(p, r);
    int64_t slot;
    if (p.slots) slot = p.slots[r];
    else slot = (p.lengths ? (int64_t)p.lengths[w.z] : p.length) + w.t;
    u32x4 out = {0, 0, 0, 0};
    if (slot >= 0 && slot < p.c.capacity) {
        const uint8_t* cb = v ? p.c.v_codes : p.c.k_codes;
        const uint8_t* sb = v ? p.c.v_scales : p.c.k_scales;
        const uint32_t codes = *(const uint32_t*)(cb + code_at(p.c, w, slot, D) + 4 * lane);
        const float scale = __uint_as_float((uint32_t)sb[scale_at(p.c, w, slot, D) + lane / 4] << 23);
        out[0] = T::template cvt<0>(codes, scale);
        out[1] = T::template cvt<1>(codes, scale);
        out[2] = T::template cvt<2>(codes, scale);
        out[3] = T::template cvt<3>(codes, scale);
    }
    typename T::elem* dst = (typename T::elem*)p.dst[v] + w.z * p.st[v][0] + w.h * p.st[v][1] + w.t * p.st[v][2];
    *(u32x4*)(dst + 8 * lane) = out;
}

template <class T>
const void* pick(bool read, int64_t d) {
    switch (d) {
        case 32: return read ? (const void*)&read_kernel<T, 32> : (const void*)&append_kernel<T, 32>;
        case 64: return read ? (const void*)&read_kernel<T, 64> : (const void*)&append_kernel<T, 64>;
        case 128: return read ? (const void*)&read_kernel<T, 128> : (const void*)&append_kernel<T, 128>;
        default: return read ? (const void*)&read_kernel<T, 256> : (const void*)&append_kernel<T, 256>;
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
    p.t = a->t;
    p.rows = a->cache.z * a->cache.h * a->t;
    const int64_t per = 256 / (a->cache.head_dim / 8);
    const int64_t blocks = (p.rows + per - 1) / per;
    if (blocks > 0x7fffffff) return RSFA_E_CACHE;
    const void* fn = a->cache.dtype == RSFA_DTYPE_BF16 ? pick<BF16>(read, a->cache.head_dim) : pick<F16>(read, a->cache.head_dim);
    void* args[] = {&p};
    if (hipLaunchKernel(fn, dim3((unsigned)blocks, 2), dim3(256), args, 0, (hipStream_t)stream) != hipSuccess)
        return RSFA_E_LAUNCH;
    return RSFA_OK;
}

}  // namespace

extern "C" {

int rsfa_cache4_append(const rsfa_cache4_rows_args* a, void* stream) { return rows_launch(a, false, stream); }
int rsfa_cache4_read(const rsfa_cache4_rows_args* a, void* stream) { return rows_launch(a, true, stream); }

}  // extern "C"
