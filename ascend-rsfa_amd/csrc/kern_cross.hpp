// Instantiations of the forward kernel for cross attention (MODE_CROSS), one list a type.  Tiles (BN, NW, OCC)
// are those of the non-causal calls (kern_d*.hip): 8 waves, 256 query rows, and 4 waves, 128 rows; at head
// dim 32 the two of 128 rows.  Head dim 64 has room for three waves a SIMD with 4 (135 registers): keys are often
// few here, and a third workgroup hides the others' starts (64 heads of 4096 tokens: 77 keys 30 -> 23 us, 512 keys
// 55 -> 46).  Bound by the matrix unit at head dim 128, 8 x 16 heads of 1024 tokens, 4096 keys 238 us, 1155 TFLOP/s, 8 x 32
// of 2048 tokens 888 us, 1238; by it and the vector unit at 64, as the non-causal calls are.
#pragma once

#include "fa_fwd_kernel.hpp"
#include "kernel_table.hpp"

#define RSFA_CROSS_ENTRY(T, DTYPE, D, BN, NW, OCC)                                       \
    {DTYPE, D, BN, NW, 0, MODE_CROSS, OCC, uses_pingpong(D, BN, NW, false, MODE_CROSS),  \
     (const void*)&fa_fwd_kernel<T, D, BN, NW, false, MODE_CROSS, OCC>, 32 * NW, 1, 32 * NW, BN}

#define RSFA_DEFINE_CROSS_LIST(NAME, T, DTYPE)                                                                        \
    RSFA_DEFINE_KERNEL_LIST(NAME, RSFA_CROSS_ENTRY(T, DTYPE, 32, 128, 4, 3), RSFA_CROSS_ENTRY(T, DTYPE, 32, 64, 4, 4), \
                            RSFA_CROSS_ENTRY(T, DTYPE, 64, 128, 8, 2), RSFA_CROSS_ENTRY(T, DTYPE, 64, 64, 4, 3),       \
                            RSFA_CROSS_ENTRY(T, DTYPE, 128, 64, 8, 2), RSFA_CROSS_ENTRY(T, DTYPE, 128, 64, 4, 2),      \
                            RSFA_CROSS_ENTRY(T, DTYPE, 256, 32, 8, 2), RSFA_CROSS_ENTRY(T, DTYPE, 256, 32, 4, 2))
