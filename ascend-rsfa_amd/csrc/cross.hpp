// What the kernels of cross attention share.
#pragma once

#include "../../include/rsfa.h"
#include "fa_fwd_kernel.hpp"

namespace rsfa {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mfma16(TypeF16::x8 a, TypeF16::x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(TypeBF16::x8 a, TypeBF16::x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The head and block of a workgroup.  Workgroups go to the 8 XCDs in turn; the blocks of a head stay on
// one (where heads divide evenly) and are neighbours in time, so that what all of them pass over is fetched into its L2 once.
__device__ __forceinline__ void head_block(int heads, int blocks, int& head, int& block) {
    int i = blockIdx.x, x = 0, step = 1;
    if (heads % 8 == 0) x = i & 7, i >>= 3, step = 8;
    const int local = i / blocks;
    block = i - local * blocks;
    head = local * step + x;
}

// Few rows: waves of a workgroup, whose tiles of 32 keys take 256 D bytes of LDS each, and waves of a SIMD.
template <int D>
struct Few {
    static constexpr int WAVES = D == 256 ? 2 : 4;
    static constexpr int OCC = D >= 128 ? 1 : 2;
};

// Sizes and types of a call (RSFA_OK or a status).
inline int cross_check(int32_t dtype, int64_t z, int64_t heads, int64_t key_heads, int64_t t, int64_t n, int64_t d) {
    if (dtype != RSFA_DTYPE_F16 && dtype != RSFA_DTYPE_BF16) return RSFA_E_DTYPE;
    if (d != 32 && d != 64 && d != 128 && d != 256) return RSFA_E_CROSS;
    if (z < 1 || key_heads < 1 || heads < 1 || heads % key_heads || t < 1 || n < 1) return RSFA_E_CROSS;
    if (z > (1 << 24) || heads > (1 << 24) || z * heads > (1 << 24) || t > (1 << 28) || n > (1 << 30) ||
        heads / key_heads * t > (1 << 28) || z * heads * t > (int64_t(1) << 40))
        return RSFA_E_CROSS;
    return RSFA_OK;
}

// Rows of 16-byte units; a tile's rows (up to 128) lie within the 32-bit offsets of the direct loads.
inline int cross_check_rows(const void* p, const int64_t st[4]) {
    if ((uintptr_t)p & 15) return RSFA_E_ALIGN;
    if (st[3] != 1) return RSFA_E_ALIGN;
    for (int i = 0; i < 3; ++i)
        if (st[i] < 0 || st[i] % 8) return RSFA_E_ALIGN;
    return (127 * st[2] + 256) * 2 < (int64_t(1) << 32) ? RSFA_OK : RSFA_E_ALIGN;
}

// Compute units of the current device (256 where none is visible).
inline int cross_cus() {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1)
        return 256;
    return n;
}

}  // namespace rsfa
