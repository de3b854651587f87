// Eviction from a 4-bit cache by accumulated weight: rsfa_cache4_claim and
// rsfa_cache4_evict (include/rsfa.h).
//
// select_kernel: one workgroup per sequence and head finds the v slots that go
// first, by weight, ties by slot.  Weights become unsigned keys of the same order,
// held in registers; the v-th smallest is found digit by digit (2048 bins in
// LDS), starting from the range that the row's keys span, so that the first
// digit already spreads them (the leading bits of a float hardly differ within a
// row).  A wave holds consecutive slots, so ranks need one exchange of counts
// between the waves and the order of atomics has no say in the result.
// gather_kernel: copies the slots that stay, 16 bytes of codes and the scale
// byte of their block a lane.
// Bound: reading 4 (weights) + 4 (positions, where some are protected) bytes a slot, and
// 2 * (D/2 + D/32) + 8 bytes in and out of each slot that is copied.
#include "cache4.hpp"

using namespace rsfa4;

namespace {

constexpr uint32_t PROTECTED = 0xffffffffu;  // above every weight's key
constexpr int DIGIT = 11, BINS = 1 << DIGIT;

struct EvictParams {
    rsfa_cache4 c, into;
    const int32_t* lengths;
    int64_t length;
    int64_t n, budget, recent, sinks;
    int32_t evict;  // 0: claim
    int32_t* out;   // claim: [bh][n]; evict: [bh][budget], the slots that stay
};

// Keys order as the weights do: -0 as 0, NaN above all others.
__device__ __forceinline__ uint32_t key_of(float w) {
    const uint32_t b = __float_as_uint(w);
    if (w != w) return 0xfffffffeu;
    if ((b & 0x7fffffffu) == 0) return 0x80000000u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <int THREADS>
struct Shared {
    uint32_t bins[BINS];
    uint32_t wave[4][THREADS / 64];
    uint32_t found[2];
};

// KPT keys a thread, wave w holding slots [w * 64 KPT, ...); KPT = 0: any number,
// read again where they are needed.
template <int THREADS, int KPT>
__global__ void __launch_bounds__(THREADS) select_kernel(EvictParams p) {
    constexpr int WAVES = THREADS / 64;
    __shared__ Shared<THREADS> sh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int bh = blockIdx.x;
    const int z = bh / (int)p.c.h, h = bh - z * (int)p.c.h;
    const int len = length_of(p.lengths, p.length, z, p.c.capacity);
    const int64_t at = z * p.c.slot_stride[0] + h * p.c.slot_stride[1];
    const float* weights = p.c.weights + at;
    const int32_t* pos = p.c.positions + at;
    const int kpt = KPT ? KPT : (int)((p.c.capacity + THREADS - 1) / THREADS);
    const int64_t seg = (int64_t)wave * 64 * kpt;
    // rounds of 64 slots of this wave that hold a slot in use
    const int rounds = (int)(seg >= len ? 0 : min((int64_t)kpt, (len - seg + 63) / 64));
    const bool guarded = p.recent > 0 || p.sinks > 0;

    // positions above `newest - recent` are protected
    int64_t old = 0x7fffffffll + 1;
    if (p.recent > 0) {
        int top = -0x7fffffff - 1;
        for (int j = 0; j < rounds; ++j) {
            const int64_t i = seg + 64 * j + lane;
            if (i < len) top = max(top, pos[i]);
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) top = max(top, __shfl_xor(top, d));
        if (lane == 0) sh.wave[0][wave] = (uint32_t)top;
        __syncthreads();
        for (int w = 0; w < WAVES; ++w) top = max(top, (int)sh.wave[0][w]);
        old = (int64_t)top - p.recent;
        __syncthreads();
    }
    auto read_key = [&](int64_t i) -> uint32_t {
        if (i >= len) return PROTECTED;
        if (guarded) {
            const int v = pos[i];
            if ((int64_t)v > old || (int64_t)v < p.sinks) return PROTECTED;
        }
        return key_of(weights[i]);
    };
    uint32_t held[KPT ? KPT : 1];
    if constexpr (KPT > 0) {
#pragma unroll
        for (int j = 0; j < KPT; ++j) held[j] = read_key(seg + 64 * j + lane);
    }
    auto each = [&](auto&& f) {
        if constexpr (KPT > 0) {
#pragma unroll
            for (int j = 0; j < KPT; ++j)
                if (j < rounds) f(held[j], seg + 64 * j + lane);
        } else {
            for (int j = 0; j < rounds; ++j) f(read_key(seg + 64 * j + lane), seg + 64 * j + lane);
        }
    };

    // candidates, and the range of their keys
    uint32_t low = PROTECTED, high = 0, count = 0;
    each([&](uint32_t k, int64_t) {
        if (k != PROTECTED) low = min(low, k), high = max(high, k), ++count;
    });
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        low = min(low, (uint32_t)__shfl_xor((int)low, d));
        high = max(high, (uint32_t)__shfl_xor((int)high, d));
        count += __shfl_xor((int)count, d);
    }
    if (lane == 0) sh.wave[0][wave] = low, sh.wave[1][wave] = high, sh.wave[2][wave] = count;
    __syncthreads();
    low = PROTECTED, high = 0, count = 0;
    for (int w = 0; w < WAVES; ++w) {
        low = min(low, sh.wave[0][w]);
        high = max(high, sh.wave[1][w]);
        count += sh.wave[2][w];
    }
    __syncthreads();

    // v slots go: those with keys below `edge`, and the first `ties` of those that have it
    const int64_t room = p.budget - len;
    const int64_t free = p.evict ? 0 : room < 0 ? 0 : min(room, p.n);
    int64_t v = p.evict ? (room < 0 ? -room : 0) : min(p.n - free, (int64_t)count);
    uint32_t edge = 0;
    int64_t ties = 0;
    if (v >= (int64_t)count) {
        if (v > 0) edge = PROTECTED, ties = v - count;
    } else if (v > 0) {
        uint32_t base = low, rest = (uint32_t)v;
        int width = high == low ? 0 : 32 - __clz((int)(high - low));
        while (width > 0) {
            const int shift = width > DIGIT ? width - DIGIT : 0;
            for (int i = threadIdx.x; i < BINS; i += THREADS) sh.bins[i] = 0;
            __syncthreads();
            each([&](uint32_t k, int64_t) {
                const uint32_t d = k - base;
                const bool in = k != PROTECTED && k >= base && (width == 32 || (d >> width) == 0);
                if (!__any(in)) return;
                const uint32_t bin = in ? d >> shift : 0;
                // (one addition where a wave's keys all share a bin, as equal weights do)
                const uint64_t who = __ballot(in);
                const int first = __ffsll((unsigned long long)who) - 1;
                const uint32_t its = (uint32_t)__shfl((int)bin, first);
                if (__ballot(in && bin == its) == who) {
                    if (lane == first) atomicAdd(&sh.bins[its], (uint32_t)__popcll(who));
                } else if (in) {
                    atomicAdd(&sh.bins[bin], 1u);
                }
            });
            __syncthreads();
            constexpr int PER = BINS / THREADS;
            uint32_t mine = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) mine += sh.bins[threadIdx.x * PER + i];
            uint32_t scan = mine;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t o = (uint32_t)__shfl_up((int)scan, d);
                if (lane >= d) scan += o;
            }
            if (lane == 63) sh.wave[3][wave] = scan;
            __syncthreads();
            uint32_t before = scan - mine;
            for (int w = 0; w < wave; ++w) before += sh.wave[3][w];
            if (before < rest && rest <= before + mine) {
                for (int i = 0; i < PER; ++i) {
                    const uint32_t b = sh.bins[threadIdx.x * PER + i];
                    if (rest <= before + b) {
                        sh.found[0] = (uint32_t)(threadIdx.x * PER + i);
                        sh.found[1] = before;
                        break;
                    }
                    before += b;
                }
            }
            __syncthreads();
            base += sh.found[0] << shift;
            rest -= sh.found[1];
            width = shift;
            __syncthreads();
        }
        edge = base;
        ties = rest;
    }

    // ranks: counts of the waves before, then along the wave
    uint32_t below = 0, same = 0;
    each([&](uint32_t k, int64_t i) {
        const bool live = i < len;
        below += __popcll(__ballot(live && k < edge));
        same += __popcll(__ballot(live && k == edge));
    });
    if (lane == 0) sh.wave[0][wave] = below, sh.wave[1][wave] = same;
    __syncthreads();
    int64_t gone = 0, seen = 0;  // that go / have the edge's key, before this round
    for (int w = 0; w < wave; ++w) gone += sh.wave[0][w], seen += sh.wave[1][w];
    gone += min(seen, ties);
    int32_t* out = p.out + (int64_t)bh * (p.evict ? p.budget : p.n);
    each([&](uint32_t k, int64_t i) {
        const bool live = i < len;
        const uint64_t lower = ((uint64_t)1 << lane) - 1;
        const uint64_t eq = __ballot(live && k == edge);
        const bool goes = live && (k < edge || (k == edge && seen + __popcll(eq & lower) < ties));
        const uint64_t who = __ballot(goes);
        const int64_t rank = gone + __popcll(who & lower);
        if (p.evict) {
            if (live && !goes) out[i - rank] = (int32_t)i;
        } else if (goes) {
            out[free + rank] = (int32_t)i;
        }
        gone += __popcll(who);
        seen += __popcll(eq);
    });
    if (!p.evict)
        for (int64_t i = threadIdx.x; i < p.n; i += THREADS) {
            if (i < free) out[i] = (int32_t)(len + i);
            else if (i >= free + v) out[i] = -1;
        }
}

template <int D>
__global__ void __launch_bounds__(256) gather_kernel(EvictParams p) {
    constexpr int LANES = D / 32;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t r = id / LANES;
    const int b = (int)(id - r * LANES);
    const int64_t bh = r / p.budget;
    if (bh >= p.c.z * p.c.h) return;
    const int64_t to = r - bh * p.budget;
    const int z = (int)(bh / p.c.h), h = (int)(bh - (int64_t)z * p.c.h);
    if (to >= length_of(p.lengths, p.length, z, p.c.capacity)) return;
    const int64_t from = p.out[r];
    const int64_t ci = z * p.c.code_stride[0] + h * p.c.code_stride[1] + from * (D / 2) + 16 * b;
    const int64_t co = z * p.into.code_stride[0] + h * p.into.code_stride[1] + to * (D / 2) + 16 * b;
    const int64_t si = z * p.c.scale_stride[0] + h * p.c.scale_stride[1] + from * LANES + b;
    const int64_t so = z * p.into.scale_stride[0] + h * p.into.scale_stride[1] + to * LANES + b;
    const u32x4 k = *(const u32x4*)(p.c.k_codes + ci), v = *(const u32x4*)(p.c.v_codes + ci);
    const uint8_t ks = p.c.k_scales[si], vs = p.c.v_scales[si];
    *(u32x4*)(p.into.k_codes + co) = k;
    *(u32x4*)(p.into.v_codes + co) = v;
    p.into.k_scales[so] = ks;
    p.into.v_scales[so] = vs;
    if (b == 0) {
        const int64_t wi = z * p.c.slot_stride[0] + h * p.c.slot_stride[1] + from;
        const int64_t wo = z * p.into.slot_stride[0] + h * p.into.slot_stride[1] + to;
        p.into.positions[wo] = p.c.positions[wi];
        if (p.into.weights) p.into.weights[wo] = p.c.weights[wi];
    }
}

int evict_launch(const rsfa_cache4_evict_args* a, bool evict, void* stream) {
    if (!a) return RSFA_E_NULL;
    if (a->struct_size != sizeof(rsfa_cache4_evict_args)) return RSFA_E_ABI;
    int st = check_cache(a->cache, true);
    if (st != RSFA_OK) return st;
    if (evict) {
        if ((st = check_cache(a->into, false)) != RSFA_OK) return st;
        if (a->into.z != a->cache.z || a->into.h != a->cache.h || a->into.head_dim != a->cache.head_dim ||
            a->into.dtype != a->cache.dtype || a->budget > a->into.capacity)
            return RSFA_E_BUDGET;
    }
    if (a->budget < 1 || a->budget > (evict ? a->into.capacity : a->cache.capacity) || a->recent < 0 || a->sinks < 0 ||
        a->recent > a->budget || a->sinks > a->budget - a->recent || (!evict && (a->n < 1 || a->n > (1 << 30))))
        return RSFA_E_BUDGET;
    if ((uintptr_t)a->lengths & 3) return RSFA_E_ALIGN;
    const int64_t bh = a->cache.z * a->cache.h;
    if (!a->out) return evict ? RSFA_E_WORKSPACE : RSFA_E_NULL;
    if ((uintptr_t)a->out & 3) return RSFA_E_ALIGN;
    if (a->out_bytes < (uint64_t)bh * (uint64_t)(evict ? a->budget : a->n) * 4) return RSFA_E_WORKSPACE;
    EvictParams p{};
    p.c = a->cache;
    if (evict) p.into = a->into;
    p.lengths = a->lengths, p.length = a->length;
    p.n = a->n, p.budget = a->budget, p.recent = a->recent, p.sinks = a->sinks;
    p.evict = evict ? 1 : 0;
    p.out = a->out;
    const int64_t c = a->cache.capacity;
    const void* fn;
    int threads = 1024;
    if (c <= 2048) fn = (const void*)&select_kernel<256, 8>, threads = 256;
    else if (c <= 8192) fn = (const void*)&select_kernel<1024, 8>;
    else if (c <= 32768) fn = (const void*)&select_kernel<1024, 32>;
    else if (c <= 65536) fn = (const void*)&select_kernel<1024, 64>;
    else fn = (const void*)&select_kernel<1024, 0>;
    const int64_t blocks = evict ? (bh * a->budget * (a->cache.head_dim / 32) + 255) / 256 : 1;
    if (blocks > 0x7fffffff) return RSFA_E_CACHE;
    void* args[] = {&p};
    if (hipLaunchKernel(fn, dim3((unsigned)bh), dim3((unsigned)threads), args, 0, (hipStream_t)stream) != hipSuccess)
        return RSFA_E_LAUNCH;
    if (!evict) return RSFA_OK;
    const int64_t d = a->cache.head_dim;
    fn = d == 32    ? (const void*)&gather_kernel<32>
         : d == 64  ? (const void*)&gather_kernel<64>
         : d == 128 ? (const void*)&gather_kernel<128>
                    : (const void*)&gather_kernel<256>;
    if (hipLaunchKernel(fn, dim3((unsigned)blocks), dim3(256), args, 0, (hipStream_t)stream) != hipSuccess)
        return RSFA_E_LAUNCH;
    return RSFA_OK;
}

}  // namespace

extern "C" {

int rsfa_cache4_claim(const rsfa_cache4_evict_args* a, void* stream) { return evict_launch(a, false, stream); }
int rsfa_cache4_evict(const rsfa_cache4_evict_args* a, void* stream) { return evict_launch(a, true, stream); }

}  // extern "C"
