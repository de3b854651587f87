// What the kernels of the 4-bit key/value cache share (format: include/rsfa.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/rsfa.h"

namespace rsfa4 {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The types a cache stands for.  The conversions take the scale from the
// exponent bits of a float and ignore its other bits, so a scale byte only has
// to be brought to bits 23 .. 30.
struct F16 {
    typedef _Float16 elem;
    typedef _Float16 x8 __attribute__((ext_vector_type(8)));
    typedef _Float16 x2 __attribute__((ext_vector_type(2)));
    static constexpr int lo = -23, hi = 13;  // scale exponents (include/rsfa.h)
    // values SEL of a byte-pair index into `codes`: byte SEL's two codes
    template <int SEL>
    static __device__ __forceinline__ uint32_t cvt(uint32_t codes, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, SEL));
    }
    static __device__ __forceinline__ f32x4 mfma(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

struct BF16 {
    typedef __bf16 elem;
    typedef __bf16 x8 __attribute__((ext_vector_type(8)));
    typedef __bf16 x2 __attribute__((ext_vector_type(2)));
    static constexpr int lo = -125, hi = 125;
    template <int SEL>
    static __device__ __forceinline__ uint32_t cvt(uint32_t codes, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, SEL));
    }
    static __device__ __forceinline__ f32x4 mfma(x8 a, x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

// Slots of sequence z in use: the length, within [0, most].
__device__ __forceinline__ int length_of(const int32_t* lengths, int64_t length, int z, int64_t most) {
    const int64_t n = lengths ? (int64_t)lengths[z] : length;
    return (int)(n < 0 ? 0 : n > most ? most : n);
}

// Sizes, pointers and strides of a cache (RSFA_OK or a status).
inline int check_cache(const rsfa_cache4& c, bool weights) {
    if (!c.k_codes || !c.k_scales || !c.v_codes || !c.v_scales || !c.positions || (weights && !c.weights))
        return RSFA_E_NULL;
    if (c.dtype != RSFA_DTYPE_F16 && c.dtype != RSFA_DTYPE_BF16) return RSFA_E_DTYPE;
    const int64_t d = c.head_dim;
    if (d != 32 && d != 64 && d != 128 && d != 256) return RSFA_E_CACHE;
    if (c.z < 1 || c.h < 1 || c.capacity < 1 || c.z > (1 << 24) || c.h > (1 << 24) || c.z * c.h > (1 << 24) ||
        c.capacity > (1 << 30))
        return RSFA_E_CACHE;
    if (((uintptr_t)c.k_codes | (uintptr_t)c.v_codes) & 15) return RSFA_E_ALIGN;
    if (((uintptr_t)c.k_scales | (uintptr_t)c.v_scales) & (d / 32 - 1)) return RSFA_E_ALIGN;
    if (((uintptr_t)c.positions | (uintptr_t)c.weights) & 3) return RSFA_E_ALIGN;
    for (int i = 0; i < 2; ++i) {
        if (c.code_stride[i] < 0 || c.scale_stride[i] < 0 || c.slot_stride[i] < 0) return RSFA_E_ALIGN;
        if (c.code_stride[i] % 16 || c.scale_stride[i] % (d / 32)) return RSFA_E_ALIGN;
    }
    return RSFA_OK;
}

// Rows q, o, k or v: 16-byte aligned, the last stride 1.
inline int check_rows(const void* p, const int64_t st[4]) {
    if ((uintptr_t)p & 15) return RSFA_E_ALIGN;
    if (st[3] != 1) return RSFA_E_ALIGN;
    for (int i = 0; i < 3; ++i)
        if (st[i] < 0 || st[i] % 8) return RSFA_E_ALIGN;
    return RSFA_OK;
}

}  // namespace rsfa4
