// Drafted tokens: which ones each sees, from their tree (rsfa_draft_tree), and keeping the accepted ones in a
// 4-bit cache (rsfa_cache4_keep); declared in include/rsfa.h.
#include "cache4.hpp"

using namespace rsfa4;

namespace {

// A token's bits are its own and its ancestors'.  By doubling: with up[i] the ancestor 2^r above token i
// and the bits of all nearer ones in row i, a round adds the row of up[i] and moves up[i] to up[up[i]], so a
// path of t tokens takes log2(t) rounds of LDS reads and not t.  One workgroup a tree, one thread a token; bound by
// the latency of a launch and of the rounds: one tree of 7 tokens 3.6 us, 32 of 25 4.6.
struct TreeParams {
    const int32_t* parents;
    int64_t stride;
    int32_t t, words;
    uint32_t* bits;
    int32_t* depths;
};

constexpr int WORDS = RSFA_DRAFT_TOKENS / 32;

__global__ void __launch_bounds__(RSFA_DRAFT_TOKENS) tree_kernel(TreeParams p) {
    __shared__ uint32_t rows[RSFA_DRAFT_TOKENS * WORDS];
    __shared__ int ups[RSFA_DRAFT_TOKENS];
    const int i = threadIdx.x;
    const bool there = i < p.t;
    uint32_t row[WORDS];
    int up = there ? p.parents[blockIdx.x * p.stride + i] : -1;
    if (up < 0 || up >= i) up = -1;  // the context's last token
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
        row[w] = (w == i / 32 ? 1u << i % 32 : 0u) | (up >= 0 && w == up / 32 ? 1u << up % 32 : 0u);
        if (there && w < p.words) rows[i * p.words + w] = row[w];
    }
    ups[i] = up;
    __syncthreads();
    for (int reach = 1; reach < p.t; reach *= 2) {
        int next = -1;
        if (up >= 0) {
            next = ups[up];
#pragma unroll
            for (int w = 0; w < WORDS; ++w)
                if (w < p.words) row[w] |= rows[up * p.words + w];
        }
        __syncthreads();
        if (up >= 0) {
#pragma unroll
            for (int w = 0; w < WORDS; ++w)
                if (w < p.words) rows[i * p.words + w] = row[w];
        }
        ups[i] = up = next;
        __syncthreads();
    }
    if (!there) return;
    int depth = -1;
#pragma unroll
    for (int w = 0; w < WORDS; ++w)
        if (w < p.words) {
            depth += __popc(row[w]);
            p.bits[((int64_t)blockIdx.x * p.t + i) * p.words + w] = row[w];
        }
    p.depths[(int64_t)blockIdx.x * p.t + i] = depth;
}

// Row j of a sequence's accepted tokens goes from slot start + tokens[j] to slot start + j.  Target slots may be
// sources of other rows, in any order, so a workgroup has all that it moves in LDS before it writes: it moves one
// of three columns (K codes, V codes, the rest) of one sequence and head, which no other touches.  Bound by the latency
// of the launch and of three loads that wait for each other (length, token, row): 5 rows of 8 heads, D = 128, 2.8 us; up to 17 of
// 64 x 8 heads, D = 256, 4.0.
struct KeepParams {
    rsfa_cache4 c;
    const int32_t *tokens, *lengths, *counts, *pos_start;
    int64_t length;
    int32_t n;
};

template <int D>
__global__ void __launch_bounds__(256) keep_kernel(KeepParams p) {
    extern __shared__ __attribute__((aligned(16))) char held[];
    const int bh = blockIdx.x;
    const int z = bh / (int)p.c.h, h = bh - z * (int)p.c.h;
    const int64_t start = length_of(p.lengths, p.length, z, p.c.capacity);
    const int rows = p.counts ? max(0, min(p.counts[z], p.n)) : p.n;
    const int32_t* tokens = p.tokens + (int64_t)z * p.n;
    // the slot that row j comes from, or -1: none, or row j has no slot to go to
    auto source = [&](int j) -> int64_t {
        const int64_t t = tokens[j];
        return t >= 0 && start + t < p.c.capacity && start + j < p.c.capacity ? start + t : -1;
    };
    if (blockIdx.y < 2) {
        constexpr int UNITS = D / 32;  // 16-byte units of a row's codes
        u32x4* const lds = (u32x4*)held;
        uint8_t* const base = (blockIdx.y ? p.c.v_codes : p.c.k_codes) + z * p.c.code_stride[0] + h * p.c.code_stride[1];
        for (int i = threadIdx.x; i < rows * UNITS; i += 256) {
            const int64_t from = source(i / UNITS);
            if (from >= 0) lds[i] = *(const u32x4*)(base + from * (D / 2) + i % UNITS * 16);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < rows * UNITS; i += 256)
            if (source(i / UNITS) >= 0) *(u32x4*)(base + (start + i / UNITS) * (D / 2) + i % UNITS * 16) = lds[i];
        return;
    }
    constexpr int W = D / 32;  // scale bytes of a row
    struct Rest {
        uint8_t k[W], v[W];
    };
    float* const lds_w = (float*)held;
    Rest* const lds_s = (Rest*)(held + p.n * 4);
    uint8_t* const ks = p.c.k_scales + z * p.c.scale_stride[0] + h * p.c.scale_stride[1];
    uint8_t* const vs = p.c.v_scales + z * p.c.scale_stride[0] + h * p.c.scale_stride[1];
    const int64_t slots = z * p.c.slot_stride[0] + h * p.c.slot_stride[1];
    for (int j = threadIdx.x; j < rows; j += 256) {
        const int64_t from = source(j);
        if (from < 0) continue;
        __builtin_memcpy(lds_s[j].k, __builtin_assume_aligned(ks + from * W, W), W);
        __builtin_memcpy(lds_s[j].v, __builtin_assume_aligned(vs + from * W, W), W);
        if (p.c.weights) lds_w[j] = p.c.weights[slots + from];
    }
    __syncthreads();
    const int64_t at = p.pos_start ? (int64_t)p.pos_start[z] : start;
    for (int j = threadIdx.x; j < rows; j += 256) {
        if (source(j) < 0) continue;
        __builtin_memcpy(__builtin_assume_aligned(ks + (start + j) * W, W), lds_s[j].k, W);
        __builtin_memcpy(__builtin_assume_aligned(vs + (start + j) * W, W), lds_s[j].v, W);
        if (p.c.weights) p.c.weights[slots + start + j] = lds_w[j];
        p.c.positions[slots + start + j] = (int32_t)(at + j);
    }
}

}  // namespace

extern "C" {

int rsfa_draft_tree(const rsfa_draft_tree_args* a, void* stream) {
    if (!a) return RSFA_E_NULL;
    if (a->struct_size != sizeof(rsfa_draft_tree_args)) return RSFA_E_ABI;
    if (!a->parents || !a->bits || !a->depths) return RSFA_E_NULL;
    if (((uintptr_t)a->parents | (uintptr_t)a->bits | (uintptr_t)a->depths) & 3) return RSFA_E_ALIGN;
    if (a->t < 1 || a->t > RSFA_DRAFT_TOKENS || a->trees < 1 || a->trees > (1 << 24) || a->parents_stride < 0) return RSFA_E_DRAFT;
    TreeParams p{a->parents, a->parents_stride, (int32_t)a->t, (int32_t)(a->t + 31) / 32, (uint32_t*)a->bits, a->depths};
    void* args[] = {&p};
    const unsigned threads = (unsigned)(a->t + 63) / 64 * 64;
    return hipLaunchKernel((const void*)&tree_kernel, dim3((unsigned)a->trees), dim3(threads), args, 0, (hipStream_t)stream) == hipSuccess
               ? RSFA_OK : RSFA_E_LAUNCH;
}

int rsfa_cache4_keep(const rsfa_cache4_keep_args* a, void* stream) {
    if (!a) return RSFA_E_NULL;
    if (a->struct_size != sizeof(rsfa_cache4_keep_args)) return RSFA_E_ABI;
    const int st = check_cache(a->cache, false);
    if (st != RSFA_OK) return st;
    if (!a->tokens) return RSFA_E_NULL;
    if (((uintptr_t)a->tokens | (uintptr_t)a->lengths | (uintptr_t)a->counts | (uintptr_t)a->pos_start) & 3) return RSFA_E_ALIGN;
    if (a->n < 1 || a->n > RSFA_DRAFT_TOKENS) return RSFA_E_DRAFT;
    KeepParams p{a->cache, a->tokens, a->lengths, a->counts, a->pos_start, a->length, (int32_t)a->n};
    void* args[] = {&p};
    const int64_t d = a->cache.head_dim;
    const void* fn = d == 32 ? (const void*)&keep_kernel<32> : d == 64 ? (const void*)&keep_kernel<64>
                   : d == 128 ? (const void*)&keep_kernel<128> : (const void*)&keep_kernel<256>;
    const size_t lds = (size_t)a->n * std::max<int64_t>(d / 2, 4 + d / 16);  // codes; or a weight and two rows of scales
    return hipLaunchKernel(fn, dim3((unsigned)(a->cache.z * a->cache.h), 3), dim3(256), args, lds, (hipStream_t)stream) == hipSuccess
               ? RSFA_OK : RSFA_E_LAUNCH;
}

}  // extern "C"
