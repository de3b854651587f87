/*
 * rsfa.h - C ABI of the MI355X (gfx950) FlashAttention-2 forward library.
 *
 * This is the only native boundary of the package.  The Python module
 * ascend_rsfa.flash_attention_forward binds it with ctypes; any other host
 * language can bind the same symbols (plain pointers, sizes and ints, no
 * torch or C++ types in any signature).
 *
 * Every entry point below replaces one piece of the reference operator
 * (Dell710000/ascend-rsfa, file ascend_rsfa/flash_attention_forward.py):
 *
 *   rsfa_attention_fwd        -> _attention.forward, lines 547-616, i.e. the
 *                                kernel launches at 565, 574, 599 and the causal
 *                                two-launch split _run_causal_split (493-541)
 *   rsfa_get_tiling           -> get_tiling(Z, H, N_CTX, HEAD_DIM, causal), 624-665
 *   rsfa_resolve_tiling       -> the (BLOCK_M, BLOCK_N) meta-parameters the
 *                                reference passes to _attn_fwd[grid] (518-519, 606-607)
 *   rsfa_get_num_compute_cores-> get_num_compute_cores(), 19-21
 *   rsfa_v8_workspace_bytes   -> (no counterpart: workspace a float8 V needs,
 *                                for the fp8_v branch of _attn_fwd_inner,
 *                                208-211; zero, the kernels read V's bytes;
 *                                kept so that callers of ABI version 5 link)
 *   rsfa_strerror             -> (no counterpart: the reference raises Python
 *                                exceptions; codes map to them in the wrapper)
 *
 * rsfa_rotary, rsfa_cache4_*, rsfa_cross_* and rsfa_draft_tree (below) have no
 * counterpart in the reference: they are what a program that serves with the
 * operator, or trains a decoder with an encoder, runs around it.
 *
 * Conventions
 *   - All tensor pointers are device pointers owned by the caller; the library
 *     never frees them.  Strides are in elements.  The last (head-dim) stride
 *     of q/k/v/o must be 1, every other stride a multiple of 8 elements (16
 *     for a float8 V) and every base pointer 16-byte aligned.  The K and V
 *     row strides (and at D = 64 and 128 the Q row stride, whose rows the
 *     8-wave tiles load the same way) must also keep BLOCK_N rows inside
 *     4 GiB: ((BLOCK_N - 1) * row_stride + max(D, 32)) * 2 < 2^32 bytes for
 *     every tile the call could run (BLOCK_N <= 128: row strides below
 *     ~16.9 M elements always pass).  RSFA_E_ALIGN otherwise.
 *   - Work is enqueued asynchronously on `stream` (a hipStream_t, NULL = the
 *     null stream).  The call returns after the launch, not after completion.
 *   - Return codes: 0 on success, a negative rsfa_status otherwise.  Invalid
 *     arguments are rejected before anything is launched.
 */
#ifndef RSFA_H_
#define RSFA_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define RSFA_ABI_VERSION 6

typedef enum rsfa_status {
    RSFA_OK          = 0,
    RSFA_E_NULL      = -1,  /* a required pointer is NULL                      */
    RSFA_E_SHAPE     = -2,  /* Z, H or N_CTX not >= 1, or too large             */
    RSFA_E_HEADDIM   = -3,  /* head_dim not in {16, 32, 64, 128, 256}           */
    RSFA_E_DTYPE     = -4,  /* dtype not one of rsfa_dtype                      */
    RSFA_E_TILE      = -5,  /* block_m/block_n invalid (see rsfa_resolve_tiling)*/
    RSFA_E_ALIGN     = -6,  /* stride / alignment contract violated             */
    RSFA_E_DEVICE    = -7,  /* HIP runtime error while querying or preparing    */
    RSFA_E_LAUNCH    = -8,  /* kernel launch failed                             */
    RSFA_E_ABI       = -9,  /* struct_size does not match this library          */
    RSFA_E_WORKSPACE = -10, /* split mode without a large enough workspace       */
    RSFA_E_SCRATCH   = -11, /* rsfa_attention_fwd_noalloc: the problem needs
                               more workspace than RSFA_NOALLOC_WORKSPACE_BYTES */
    RSFA_E_ROTARY    = -12, /* rsfa_rotary: rotary_dim odd, < 2 or > head_dim   */
    RSFA_E_CACHE     = -13, /* a cache or a call on one is out of its range: see
                               rsfa_cache4                                      */
    RSFA_E_BUDGET    = -14, /* claim / evict: budget, recent, sinks or n         */
    RSFA_E_CROSS     = -16, /* cross attention: sizes or heads                  */
    RSFA_E_DRAFT     = -15  /* drafted tokens: more than RSFA_DRAFT_TOKENS, or
                               an option that a tree does not go with           */
} rsfa_status;

typedef enum rsfa_dtype {
    RSFA_DTYPE_F16  = 0,         /* q, k, v, o float16                         */
    RSFA_DTYPE_BF16 = 1,         /* q, k, v, o bfloat16                        */
    RSFA_DTYPE_F16_V8E5M2 = 2,   /* q, k, o float16; v float8 e5m2 (OCP: sign,
                                    5 exponent bits, bias 15, 2 mantissa bits).
                                    P is rounded to e5m2 for P.V and the row
                                    sums add the unrounded P, as the reference's
                                    fp8_v branch does (208-211, 217).  The
                                    kernels read V's bytes and run P.V on the
                                    e5m2 MFMA at every head dim (no
                                    workspace) */
    RSFA_DTYPE_F32 = 3           /* float32: rsfa_rotary only                   */
} rsfa_dtype;

/* flags (bit set) */
#define RSFA_FLAG_STATIC_SCHEDULE 0x1u /* grid-stride task order instead of the
                                          dynamic atomic-ticket queue            */
#define RSFA_FLAG_CAUSAL_SPLIT    0x2u /* causal only: two launches, mask-free
                                          prefix then masked diagonal, with the
                                          (m, l, acc) state handed over in fp32
                                          through `workspace` (reference
                                          493-541)                              */
#define RSFA_FLAG_EXACT_TILE      0x4u /* a request (block_m, block_n) runs the
                                          compiled tile nearest to it, never a
                                          key-split variant of the tile (see
                                          block_m); overrides TILE_HINT         */
#define RSFA_FLAG_TILE_HINT       0x8u /* a valid request is only checked, and
                                          the tile rsfa_get_tiling picks for
                                          the shape runs                        */
#define RSFA_FLAG_SINGLE_BLOCKS   0x10u /* causal: one query block per task
                                          instead of the pairs (nmb-1-i, i) the
                                          library uses when they fill whole
                                          rounds of the grid; same results,
                                          bit for bit (a scheduling knob)       */

typedef struct rsfa_fwd_args {
    uint32_t    struct_size;  /* = sizeof(rsfa_fwd_args)                        */
    int32_t     dtype;        /* rsfa_dtype of q, k, v and o                    */
    const void *q;            /* [Z, H, N_CTX, D]                               */
    const void *k;            /* [Z, H, N_CTX, D]                               */
    const void *v;            /* [Z, H, N_CTX, D]                               */
    void       *o;            /* [Z, H, N_CTX, D], same dtype as q              */
    float      *lse;          /* optional [Z, H, N_CTX] fp32, natural-log
                                 logsumexp of the scaled scores (the reference's
                                 M = m + ln(l), 400-403); NULL = not written    */
    void       *workspace;    /* split mode: the split state
                                 (rsfa_split_workspace_bytes)                  */
    uint64_t    workspace_bytes;
    int64_t     z, h, n_ctx, head_dim;
    int64_t     q_stride[4];  /* element strides of dims (Z, H, N_CTX, D)       */
    int64_t     k_stride[4];
    int64_t     v_stride[4];
    int64_t     o_stride[4];
    float       sm_scale;     /* multiplies q.k before the softmax              */
    int32_t     causal;       /* 0/1: key n visible to query m iff n <= m       */
    int32_t     block_m;      /* requested BLOCK_M; 0 (with block_n 0) = no
                                 request, the tile rsfa_get_tiling picks runs.
                                 A request is checked against the reference's
                                 rules (RSFA_E_TILE otherwise) and, like the
                                 reference's BLOCK_M/BLOCK_N meta-parameters,
                                 selects the tile: the compiled one nearest to
                                 it runs (rsfa_resolve_tiling), unless
                                 RSFA_FLAG_TILE_HINT.  Split mode sizes its
                                 workspace with the BLOCK_M that runs.  Where
                                 the tile search answers a 128-row tile for a
                                 grid that does not fill the chip, a fused
                                 launch of it may split each task's keys over
                                 its wave groups (on 128 or 64 rows), unless
                                 RSFA_FLAG_EXACT_TILE                        */
    int32_t     block_n;      /* requested BLOCK_N (see block_m)                */
    uint32_t    flags;        /* RSFA_FLAG_*                                    */
} rsfa_fwd_args;

/* Fused FlashAttention-2 forward: o = softmax(q k^T * sm_scale [+ causal mask]) v.
 * Replaces _attention.forward (flash_attention_forward.py:547-616). */
int rsfa_attention_fwd(const rsfa_fwd_args *args, void *stream);

/* Workspace rsfa_attention_fwd_noalloc has for the split state (its fixed
 * per-device buffer holds 4 KiB of queue counters besides). */
#define RSFA_NOALLOC_WORKSPACE_BYTES (16u << 20)

/* rsfa_attention_fwd without any allocation.  It has no counterpart in the
 * reference: it is for callers that cannot allocate device memory (code under
 * HIP graph capture, tight serving loops, harnesses that forbid hipMalloc).
 * Same arguments, kernels and results as rsfa_attention_fwd, except that
 * `workspace`/`workspace_bytes` are ignored: the queue counters and the
 * workspace (the split state) live in one fixed
 * buffer per device, a static device array of RSFA_NOALLOC_WORKSPACE_BYTES
 * + 4 KiB that the device holds until the process ends.  Problems that need
 * more workspace fail with RSFA_E_SCRATCH before any device work.  The first
 * call on a device looks the buffer up (hipGetSymbolAddress); a call with more
 * tasks than workgroups clears its counters with a small kernel on `stream`
 * before the launch that takes them.  All calls on one
 * device share the buffer: calls that overlap in time on one device (other
 * streams, concurrent graph replays) race and must be serialised by the
 * caller. */
int rsfa_attention_fwd_noalloc(const rsfa_fwd_args *args, void *stream);

/* Bytes of fp32 workspace RSFA_FLAG_CAUSAL_SPLIT needs for this problem and
 * the BLOCK_M that runs (rsfa_resolve_tiling of the request, or
 * rsfa_get_tiling's without one / under RSFA_FLAG_TILE_HINT): state[2, Z, H,
 * NBM, BM] (row max in exp2 units, row sum), as the reference allocates at
 * 501, then the un-normalised accumulator [Z, H, NBM, BM, head_dim] in fp32,
 * which the reference instead rounds to the input dtype into O (353).
 * 0 for invalid sizes. */
uint64_t rsfa_split_workspace_bytes(int64_t z, int64_t h, int64_t n_ctx,
                                    int64_t head_dim, int32_t block_m);

/* Bytes of workspace a float8 V (RSFA_DTYPE_F16_V8E5M2) needs: 0 (the kernels
 * read the float8 bytes at every head dim).  ABI version 5 placed an fp16
 * copy of V at head dims 16 and 32 here, before the split state; version 6
 * has none, and the split state starts at the workspace's first byte. */
uint64_t rsfa_v8_workspace_bytes(int64_t z, int64_t h, int64_t n_ctx,
                                 int64_t head_dim);

/* Tile search for gfx950 (replaces the lookup table get_tiling, 624-665):
 * writes the (BLOCK_M, BLOCK_N) rsfa_attention_fwd runs for the shape on the
 * current device (planned for its CU count; for a 256-CU MI355X where no
 * device is visible).  Never fails for a valid shape. */
int rsfa_get_tiling(int64_t z, int64_t h, int64_t n_ctx, int64_t head_dim,
                    int32_t causal, int32_t dtype, int32_t *block_m,
                    int32_t *block_n);

/* Maps a caller-requested (BLOCK_M, BLOCK_N) to the compiled instantiation
 * a launch with that request runs (the nearest compiled tile; log distance
 * in BLOCK_M and BLOCK_N, ties to the larger BLOCK_N).
 * Requests follow the reference's rules (powers of two,
 * 16 <= BLOCK <= 512, BLOCK_M*BLOCK_N <= 65536, causal needs
 * BLOCK_N <= BLOCK_M, which the reference silently breaks on, see
 * benchmarks/run_correctness_test.py:24-25).  Returns RSFA_E_TILE otherwise. */
int rsfa_resolve_tiling(int64_t head_dim, int32_t causal, int32_t dtype,
                        int32_t req_block_m, int32_t req_block_n,
                        int32_t *block_m, int32_t *block_n);

/* Number of compute units of `device` (-1 = current device); replaces
 * get_num_compute_cores (19-21).  Negative rsfa_status on error. */
int rsfa_get_num_compute_cores(int device);

/* ------------------------------------------------------------------------
 * Rotary positions.
 *
 * The first rotary_dim values of every head are R/2 pairs (R = rotary_dim):
 * (x_i, x_(i+R/2)), or with RSFA_ROTARY_INTERLEAVED (x_2i, x_(2i+1)).  Pair i
 * of the token at position p is turned by the angle 2 pi p turns[i] and scaled
 * by `amplitude`; the other values are copied.  RSFA_ROTARY_INVERSE turns
 * back (and scales by `amplitude` all the same): the gradient of the forward
 * call.  One or two tensors (q and k) of one dtype in one launch; y[i] may be
 * x[i] with the same strides (in place), but not overlap it otherwise.
 * Strides are in elements, the last one 1; any alignment that the element
 * type has (16-byte rows take wide loads).  Angles are reduced in 64 bits:
 * their error is below 2^-52 of the angle and 2^-25 of a turn.
 * ------------------------------------------------------------------------ */
#define RSFA_ROTARY_INTERLEAVED 0x1u
#define RSFA_ROTARY_INVERSE     0x2u
#define RSFA_ROTARY_POS64       0x4u /* positions are int64 instead of int32 */

typedef struct rsfa_rotary_args {
    uint32_t      struct_size;    /* = sizeof(rsfa_rotary_args)                */
    int32_t       dtype;          /* RSFA_DTYPE_F16, _BF16 or _F32             */
    const void   *x[2];           /* [Z, heads[i], N, D]; x[1] may be NULL     */
    void         *y[2];
    int64_t       z, n, head_dim, rotary_dim;
    int64_t       heads[2];
    int64_t       x_stride[2][4]; /* element strides of dims (Z, H, N, D)      */
    int64_t       y_stride[2][4];
    const void   *positions;      /* device, or NULL: token n is at start + n  */
    int64_t       pos_stride[2];  /* of dims (Z, N) of positions, in elements  */
    int64_t       start;
    const double *turns;          /* device, [rotary_dim / 2]: turns a position */
    float         amplitude;
    uint32_t      flags;          /* RSFA_ROTARY_*                              */
} rsfa_rotary_args;

int rsfa_rotary(const rsfa_rotary_args *args, void *stream);

/* ------------------------------------------------------------------------
 * A key/value cache held in 4 bits.
 *
 * A row (one token's key or value of one head) is head_dim / 2 bytes of codes
 * and head_dim / 32 scale bytes.  Each 32 values share a scale byte b, which
 * stands for 2^(b - 127); 255 makes the block NaN.  A code is a sign bit (8) and
 * the index of 0, 0.5, 1, 1.5, 2, 3, 4, 6; byte j of a row holds value 2j in its low
 * and value 2j + 1 in its high bits (the e2m1 elements and e8m0 scales of the
 * OCP microscaling formats).  Written rows take the smallest scale of
 * which no value of the block is more than 7, within the exponents -23 .. 13
 * (float16) or -125 .. 125 (bfloat16), whose values all exist in the type:
 * values are rounded to the nearest code, ties to the even index, and end at 6
 * scales; a block that holds an infinity or a NaN is stored as NaN.  Scale
 * bytes of slots in use are expected to be of that range, or 255.
 *
 * Sequences and heads are [z, h]; each has `capacity` slots, whose rows lie
 * densely: slot s of (z, h) is at z * stride[0] + h * stride[1] + s * row, with
 * strides in elements of the buffer.  code_stride is that of k_codes and
 * v_codes, scale_stride of both scale buffers, slot_stride of positions and
 * weights.  Code buffers are 16-byte aligned with strides that are multiples
 * of 16; scale buffers aligned to head_dim / 32 bytes, with strides that are
 * multiples of it.
 *
 * Lengths say how many slots of a sequence are in use: `lengths` (device,
 * int32 [z]) or, where it is NULL, `length` for all.  Values outside
 * [0, capacity] are taken as its ends by the kernels.
 * ------------------------------------------------------------------------ */
typedef struct rsfa_cache4 {
    uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
    int32_t *positions; /* position of each slot's token                       */
    float   *weights;   /* accumulated attention weight of each slot, or NULL   */
    int64_t  z, h, capacity, head_dim; /* head_dim: 32, 64, 128 or 256          */
    int64_t  code_stride[2], scale_stride[2], slot_stride[2];
    int32_t  dtype;     /* RSFA_DTYPE_F16 or _BF16: of the rows written and read */
    int32_t  reserved;  /* 0 */
} rsfa_cache4;

/* append: writes the rows k, v [z, h, t, head_dim].  Token i of sequence z goes
 * to slot lengths[z] + i, or with `slots` (device, int32 [z, h, t], dense) to
 * slots[z, h, i]; tokens i >= counts[z] (device, int32 [z], or NULL) and
 * slots outside [0, capacity) are left out; where `slots` names a slot twice
 * the last token has it (more than 96 tokens take four launches for that).  The slot's position becomes pos_start[z] + i (NULL:
 * lengths[z] + i), its weight 0.
 * read: the values of slots start[z] + i (NULL: start0 + i), or slots[z, h, i],
 * into k, v; rows outside [0, capacity) read as 0. */
typedef struct rsfa_cache4_rows_args {
    uint32_t       struct_size; /* = sizeof(rsfa_cache4_rows_args)             */
    uint32_t       reserved;    /* 0 */
    rsfa_cache4    cache;
    void          *k, *v;       /* either may be NULL in a read                */
    int64_t        t;
    int64_t        k_stride[4], v_stride[4]; /* elements; rows 16-byte aligned */
    const int32_t *lengths;     /* append: the lengths; read: the first slots   */
    int64_t        length;
    const int32_t *slots;
    const int32_t *counts;      /* append only */
    const int32_t *pos_start;   /* append only */
} rsfa_cache4_rows_args;

int rsfa_cache4_append(const rsfa_cache4_rows_args *args, void *stream);
int rsfa_cache4_read(const rsfa_cache4_rows_args *args, void *stream);

/* attend: o = softmax(q k^T sm_scale) v over the slots in use; query head i
 * reads key head i / (heads / cache.h).  With `causal` query token i of sequence
 * z sees the slots whose position is at most pos_start[z] + i (NULL:
 * length - count + i, with the sequence's count of tokens).  Rows i >= counts[z],
 * and rows that see no slot, give 0 (lse -inf); so do rows whose visible scores are
 * all -inf (an infinite q), as hidden scores are.  With `accumulate` the weights
 * of the slots grow by the softmax weights that all rows of the call gave them.
 * Scores, sums, lse and the slots' weights are in 32 bits; for the product with v a softmax
 * weight is rounded to the cache's type (half a step), as o is.
 * Lengths above max_length (0: the capacity) are taken as max_length.  o must not
 * overlap q; calls that accumulate into one cache must not overlap in time.
 * Workspace: rsfa_cache4_attend_workspace_bytes of the same arguments (its
 * contents need not outlive the call's kernels). */
typedef struct rsfa_cache4_attend_args {
    uint32_t       struct_size; /* = sizeof(rsfa_cache4_attend_args)           */
    int32_t        causal;
    rsfa_cache4    cache;
    const void    *q;           /* [z, heads, t, head_dim], the cache's dtype  */
    void          *o;
    float         *lse;         /* [z, heads, t], dense, or NULL               */
    int64_t        heads, t;
    int64_t        q_stride[4], o_stride[4];
    const int32_t *lengths;
    int64_t        length, max_length;
    const int32_t *counts, *pos_start;
    float          sm_scale;
    int32_t        accumulate;
    void          *workspace;   /* 16-byte aligned */
    uint64_t       workspace_bytes;
} rsfa_cache4_attend_args;

int rsfa_cache4_attend(const rsfa_cache4_attend_args *args, void *stream);
uint64_t rsfa_cache4_attend_workspace_bytes(const rsfa_cache4_attend_args *args);

/* Eviction by accumulated weight.  A slot in use is protected when its position
 * is less than `sinks` or among the last `recent` up to the sequence and head's
 * largest.  Slots go in order of their weight, the lowest first, ties by the
 * lowest slot (a NaN weight counts as the largest; -0 as 0).
 * claim: out [z, h, n] (int32, dense): the slots for each sequence's next n
 * tokens: those from lengths[z] up to `budget`, then the unprotected slots that
 * go first, in order of slot; -1 where there is none.
 * evict: copies to `into` (same z, h, head_dim and dtype; no memory in common) the
 * slots that stay when the first max(0, lengths[z] - budget) go (protected ones
 * after all others), in order of slot, to its slots 0, 1, ...; other slots of `into`
 * keep what they hold.
 * Workspace: rsfa_cache4_evict_workspace_bytes of the same arguments (evict: 1
 * for evict, 0 for claim; 0 bytes for claims in caches of up to 32768 slots). */
typedef struct rsfa_cache4_evict_args {
    uint32_t       struct_size; /* = sizeof(rsfa_cache4_evict_args)            */
    uint32_t       reserved;    /* 0 */
    rsfa_cache4    cache;
    rsfa_cache4    into;        /* evict only                                  */
    const int32_t *lengths;
    int64_t        length;
    int64_t        n;           /* claim only                                  */
    int64_t        budget, recent, sinks;
    int32_t       *out;         /* claim only: the slots                       */
    void          *workspace;   /* 16-byte aligned */
    uint64_t       workspace_bytes;
} rsfa_cache4_evict_args;

int rsfa_cache4_claim(const rsfa_cache4_evict_args *args, void *stream);
int rsfa_cache4_evict(const rsfa_cache4_evict_args *args, void *stream);
uint64_t rsfa_cache4_evict_workspace_bytes(const rsfa_cache4_evict_args *args, int32_t evict);

/* ------------------------------------------------------------------------
 * Cross attention: o = softmax(q k^T sm_scale) v over keys of another length.
 *
 * q, o [z, heads, t, head_dim], k, v [z, key_heads, n, head_dim] of one dtype (float16 or
 * bfloat16); query head i reads key head i / (heads / key_heads).  With `lengths` (device, int32 [z];
 * values outside [0, n] are taken as its ends) a sequence has its first lengths[z] keys; the others
 * are not read.  A sequence without keys gives 0 (lse -inf).  Strides as everywhere;
 * a stride of 0 repeats q, k or v.  Scores, sums, lse and accumulators are in 32 bits; softmax
 * weights are rounded to the dtype for the product with v, as o is.
 * Workspace: rsfa_cross_fwd_workspace_bytes of the same arguments (its contents need not outlive the
 * call's kernels).
 * ------------------------------------------------------------------------ */
typedef struct rsfa_cross_args {
    uint32_t       struct_size; /* = sizeof(rsfa_cross_args)                   */
    int32_t        dtype;       /* RSFA_DTYPE_F16 or _BF16                      */
    const void    *q, *k, *v;
    void          *o;
    float         *lse;         /* [z, heads, t], dense, or NULL: natural log   */
    int64_t        z, heads, key_heads, t, n, head_dim; /* head_dim: 32, 64, 128, 256 */
    int64_t        q_stride[4], k_stride[4], v_stride[4], o_stride[4];
    const int32_t *lengths;     /* or NULL: n keys of all                      */
    float          sm_scale;
    uint32_t       reserved;    /* 0 */
    void          *workspace;   /* 16-byte aligned */
    uint64_t       workspace_bytes;
} rsfa_cross_args;

int rsfa_cross_fwd(const rsfa_cross_args *args, void *stream);
uint64_t rsfa_cross_fwd_workspace_bytes(const rsfa_cross_args *args);

/* Its gradients, from o and lse of the forward call, the gradient of o and, or NULL, of lse
 * ([z, heads, t], dense).  A gradient whose pointer is NULL is not computed.  Gradients are whole:
 * those of k and v are summed over the query heads of a group, and 0 for keys past a length.  Softmax weights
 * and their gradients are rounded to the dtype for the products with rows; sums are in 32 bits, each in one order, so
 * that a call gives the same bits each time.  The gradients' rows must not meet each other or an input. */
typedef struct rsfa_cross_bwd_args {
    uint32_t       struct_size; /* = sizeof(rsfa_cross_bwd_args)               */
    int32_t        dtype;
    const void    *q, *k, *v, *o;
    const float   *lse;
    const void    *grad_o;
    const float   *grad_lse;
    void          *grad_q, *grad_k, *grad_v;
    int64_t        z, heads, key_heads, t, n, head_dim;
    int64_t        q_stride[4], k_stride[4], v_stride[4], o_stride[4];
    int64_t        grad_o_stride[4], grad_q_stride[4], grad_k_stride[4], grad_v_stride[4];
    const int32_t *lengths;
    float          sm_scale;
    uint32_t       reserved;    /* 0 */
    void          *workspace;   /* 16-byte aligned */
    uint64_t       workspace_bytes;
} rsfa_cross_bwd_args;

int rsfa_cross_bwd(const rsfa_cross_bwd_args *args, void *stream);
uint64_t rsfa_cross_bwd_workspace_bytes(const rsfa_cross_bwd_args *args);

/* ------------------------------------------------------------------------
 * Drafted tokens.
 *
 * A program that drafts appends t tokens that may follow each sequence's context to its cache,
 * attends with all of them at once, and keeps those that it accepts.  The drafted tokens of a
 * sequence are its last slots in use, in order; which of them a token sees is a row of
 * (t + 31) / 32 words: token j where bit j % 32 of word j / 32 is set.
 * ------------------------------------------------------------------------ */
#define RSFA_DRAFT_TOKENS 512

/* The rows of trees: token i sees itself and its ancestors.  parents[i] is an
 * earlier token, or anything else: token i follows the context's last token.
 * depths[i] counts the ancestors: the token's position is the context's
 * length + depths[i]. */
typedef struct rsfa_draft_tree_args {
    uint32_t       struct_size; /* = sizeof(rsfa_draft_tree_args)              */
    uint32_t       reserved;    /* 0 */
    const int32_t *parents;     /* device, [trees, t], rows dense              */
    int64_t        parents_stride;
    int64_t        trees, t;    /* t: 1 .. RSFA_DRAFT_TOKENS                    */
    int32_t       *bits;        /* device, [trees, t, (t + 31) / 32], dense     */
    int32_t       *depths;      /* device, [trees, t], dense                   */
} rsfa_draft_tree_args;

int rsfa_draft_tree(const rsfa_draft_tree_args *args, void *stream);

/* rsfa_cache4_attend over a context and drafted tokens: lengths count both, the
 * t tokens (counts[z] of them) being the last slots in use.  Token i sees all slots before
 * them, and drafted token j < counts[z] where row i of `bits` has it; positions and `causal`
 * are not looked at.  `bits`: device, [t, words] for each sequence, bits_stride elements
 * apart (0: one for all).  accumulate must be 0 and pos_start NULL.  Workspace:
 * rsfa_cache4_attend_tree_workspace_bytes of the same arguments. */
int rsfa_cache4_attend_tree(const rsfa_cache4_attend_args *args, const int32_t *bits,
                            int64_t bits_stride, void *stream);
uint64_t rsfa_cache4_attend_tree_workspace_bytes(const rsfa_cache4_attend_args *args);

/* keep: row j < counts[z] (NULL: n) of drafted token tokens[z, j] goes from slot
 * lengths[z] + tokens[z, j] to slot lengths[z] + j (lengths: the contexts), with its weight, and
 * takes the position pos_start[z] + j (NULL: lengths[z] + j).  All rows are read before one is
 * written.  Tokens below 0 or past the cache leave slot lengths[z] + j as it is. */
typedef struct rsfa_cache4_keep_args {
    uint32_t       struct_size; /* = sizeof(rsfa_cache4_keep_args)             */
    uint32_t       reserved;    /* 0 */
    rsfa_cache4    cache;
    const int32_t *tokens;      /* device, [z, n], dense                       */
    int64_t        n;           /* 1 .. RSFA_DRAFT_TOKENS                       */
    const int32_t *lengths;
    int64_t        length;
    const int32_t *counts, *pos_start;
} rsfa_cache4_keep_args;

int rsfa_cache4_keep(const rsfa_cache4_keep_args *args, void *stream);

/* Static string for a status code. */
const char *rsfa_strerror(int status);

/* RSFA_ABI_VERSION the library was built with. */
int rsfa_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* RSFA_H_ */
