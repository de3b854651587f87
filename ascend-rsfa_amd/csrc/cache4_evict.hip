// Eviction from a 4-bit cache by accumulated weight: rsfa_cache4_claim and
// rsfa_cache4_evict (include/rsfa.h).
//
// Which slots go: weights become unsigned keys of the same order, and the v-th smallest
// of a row (a sequence and head) is found digit by digit, 2048 bins in LDS, from the
// range that the row's keys span, so that the first digit already spreads them
// (the leading bits of a float hardly differ within a row); once a bin holds at most
// 256 keys, they are ranked directly, each against all.  Up to 32768 slots a workgroup does it for
// a row, with the keys in registers; longer rows are cut into parts, whose workgroups
// meet between four launches (survey, histogram, collect, choose).  The order of
// atomics has no say in the result: they only count, and lists are only counted.
// gather_kernel copies the slots that stay, 16 bytes of codes and the scale byte of
// their block a lane.
// Bound: reading 4 (weights) + 4 (positions, where some are protected) bytes a slot, and
// 2 * (D/2 + D/32) + 8 bytes in and out of each slot that is copied.  In practice by
// latency: one slot of 2048 for 256 rows 6 us; 4096 slots of 64 rows 9.5 (their bytes: 0.4);
// and by the instructions of one workgroup, some 0.75 us for every 1024 slots beyond 8192: 16384 slots of 32
// rows 15 us, 32768 25, of 256 rows 18 and 32 (in four launches 32 and 33, 49 and 96);
// 65521 of 8 rows 37 in four launches (64 keys a thread do not fit the registers: 123).
// The copy of 65520 slots at D = 256 takes 9 us, 4 TB/s.
#include "cache4.hpp"

using namespace rsfa4;

namespace {

constexpr uint32_t PROTECTED = 0xffffffffu;  // above every weight's key
constexpr int DIGIT = 11, BINS = 1 << DIGIT;
constexpr int RANKED = 256;  // keys that are ranked directly

struct EvictParams {
    rsfa_cache4 c, into;
    const int32_t* lengths;
    int64_t length;
    int64_t n, budget, recent, sinks;
    int32_t evict;  // 0: claim
    int32_t* out;   // claim: [bh][n]; evict: [bh][budget], the slots that stay
    // rows in parts
    int32_t parts, part;  // parts of a row, slots of a part (a multiple of 256)
    int4* survey;         // [bh][parts]: largest position, smallest and largest key of the slots in use
    uint32_t* hist;       // [bh][parts][BINS]
    uint4* found;         // [bh]: the edge's bin, keys below it, keys in it, unprotected keys in all
    uint32_t* listed;     // [bh]: keys listed so far
    int4* counts;         // [bh][parts]: keys below the edge's bin, keys in it, and where they are listed
    uint32_t* list;       // [bh][parts * part]: the keys in it, a part's together
};

// Keys order as the weights do: -0 as 0, NaN above all others.
__device__ __forceinline__ uint32_t key_of(float w) {
    const uint32_t b = __float_as_uint(w);
    if (w != w) return 0xfffffffeu;
    if ((b & 0x7fffffffu) == 0) return 0x80000000u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// What every workgroup of a row starts from.
struct Row {
    int bh, z, h, len;
    const float* weights;
    const int32_t* pos;
    bool guarded;
};

__device__ __forceinline__ Row row_of(const EvictParams& p, int bh) {
    Row r;
    r.bh = bh;
    r.z = bh / (int)p.c.h, r.h = bh - r.z * (int)p.c.h;
    r.len = __builtin_amdgcn_readfirstlane(length_of(p.lengths, p.length, r.z, p.c.capacity));
    const int64_t at = r.z * p.c.slot_stride[0] + r.h * p.c.slot_stride[1];
    r.weights = p.c.weights + at;
    r.pos = p.c.positions + at;
    r.guarded = p.recent > 0 || p.sinks > 0;
    return r;
}

// How many slots go, of `count` unprotected ones; `free`: slots a claim takes first.
__device__ __forceinline__ int64_t victims(const EvictParams& p, int len, int64_t count, int64_t& free) {
    const int64_t room = p.budget - len;
    free = p.evict ? 0 : room < 0 ? 0 : min(room, p.n);
    return p.evict ? (room < 0 ? -room : 0) : min(p.n - free, count);
}

template <int THREADS>
struct Shared {
    uint32_t bins[BINS];
    uint32_t wave[4][THREADS / 64];
    uint32_t found[3];
    uint32_t listed;
    alignas(16) uint32_t list[RANKED];
};

// Adds a wave's keys to the bins; one addition where they all share one, as equal weights do.
template <int THREADS>
__device__ __forceinline__ void count_key(Shared<THREADS>& sh, bool in, uint32_t bin, int lane) {
    bin = in ? bin : BINS;
    const uint32_t its = (uint32_t)__builtin_amdgcn_readfirstlane((int)bin);
    if (__ballot(bin == its) == ~(uint64_t)0) {
        if (its != BINS && lane == 0) atomicAdd(&sh.bins[its], 64u);
    } else if (in) {
        atomicAdd(&sh.bins[bin], 1u);
    }
}

// The bin that the rest-th counted key is in: found = {bin, keys before it, keys in it}.
// `bin_at(i)`: the count of bin i.  Ends with a barrier.
template <int THREADS, class F>
__device__ __forceinline__ void find_bin(Shared<THREADS>& sh, uint32_t rest, int lane, int wave, F&& bin_at) {
    constexpr int PER = BINS / THREADS;
    uint32_t c[PER], mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) mine += c[i] = bin_at(threadIdx.x * PER + i);
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
        bool done = false;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (!done && rest <= before + c[i]) {
                sh.found[0] = (uint32_t)(threadIdx.x * PER + i);
                sh.found[1] = before;
                sh.found[2] = c[i];
                done = true;
            }
            before += c[i];
        }
    }
    __syncthreads();
}

// The rest-th smallest of the c <= RANKED keys of sh.list (complete, with a barrier since): edge,
// and how many of its equals count.
template <int THREADS>
__device__ __forceinline__ void rank_listed(Shared<THREADS>& sh, uint32_t c, uint32_t rest, uint32_t& edge, int64_t& ties) {
    static_assert(THREADS >= RANKED, "a thread takes a key");
    if (threadIdx.x < c) {
        const uint32_t key = sh.list[threadIdx.x];
        uint32_t less = 0, same = 0;
        for (uint32_t j = 0; j < c; j += 4) {
            const u32x4 o = *(const u32x4*)&sh.list[j];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                less += j + i < c && o[i] < key;
                same += j + i < c && o[i] == key;
            }
        }
        // (all keys that satisfy this are equal)
        if (less < rest && rest <= less + same) sh.found[0] = key, sh.found[1] = rest - less;
    }
    __syncthreads();
    edge = sh.found[0];
    ties = sh.found[1];
}

// The v-th smallest key of those `each` gives (v >= 1, below their number), which all lie in
// [low, high]: edge, and the count `ties` of its equals that go.
template <int THREADS, class E>
__device__ __forceinline__ void search(Shared<THREADS>& sh, E&& each, uint32_t low, uint32_t high, uint32_t v, int lane,
                                       int wave, uint32_t& edge, int64_t& ties) {
    uint32_t base = low, rest = v;
    int width = high == low ? 0 : 32 - __clz((int)(high - low));
    while (width > 0) {
        const int shift = width > DIGIT ? width - DIGIT : 0;
        for (int i = threadIdx.x; i < BINS; i += THREADS) sh.bins[i] = 0;
        if (threadIdx.x == 0) sh.listed = 0;
        __syncthreads();
        // (the largest key bounds the bins too: protected ones lie above it, and keys below base wrap around)
        auto last = [&](int w) { return min(high - base, w == 32 ? 0xffffffffu : (1u << w) - 1); };
        uint32_t limit = last(width);
        each([&](uint32_t k) { count_key(sh, k - base <= limit, (k - base) >> shift, lane); });
        __syncthreads();
        find_bin(sh, rest, lane, wave, [&](int i) { return sh.bins[i]; });
        base += sh.found[0] << shift;
        rest -= sh.found[1];
        width = shift;
        const uint32_t c = sh.found[2];
        if (width > 0 && c <= RANKED) {
            limit = last(width);
            each([&](uint32_t k) {
                if (k - base <= limit) sh.list[atomicAdd(&sh.listed, 1u)] = k;
            });
            __syncthreads();  // (found is read by all before it is written again)
            rank_listed(sh, c, rest, edge, ties);
            return;
        }
        __syncthreads();
    }
    edge = base;
    ties = rest;
}

// Writes a wave's slots: keys below `edge` go, and of those that have it as many as
// `ties` leaves; gone and seen count the slots before that go and that have the edge's key.
struct Writer {
    const EvictParams& p;
    int32_t* out;
    uint32_t free, ties, gone, seen, edge;
    int len;
    static __device__ __forceinline__ uint32_t before(uint64_t mask, uint32_t base) {
        return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, base));
    }
    __device__ __forceinline__ void operator()(uint32_t k, uint32_t i) {
        const bool live = i < (uint32_t)len;
        bool goes = live && k < edge;
        const uint64_t eq = __ballot(live && k == edge);
        if (eq) {
            goes |= live && k == edge && before(eq, seen) < ties;
            seen += __popcll(eq);
        }
        const uint64_t who = __ballot(goes);
        if (p.evict) {
            if (live && !goes) out[i - before(who, gone)] = (int32_t)i;
        } else if (goes) {
            out[before(who, free + gone)] = (int32_t)i;
        }
        gone += __popcll(who);
    }
};

// Keys of the slots first + 64 j + lane; positions above `old` are protected.
template <int KPT>
__device__ __forceinline__ void hold_keys(const Row& r, int64_t first, int64_t old, int64_t sinks, int lane, uint32_t* held) {
    int v[KPT];
    float w[KPT];
#pragma unroll
    for (int j = 0; j < KPT; ++j) {
        const int64_t i = first + 64 * j + lane;
        v[j] = r.guarded && i < r.len ? r.pos[i] : -0x7fffffff - 1;
        w[j] = i < r.len ? r.weights[i] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < KPT; ++j) {
        const bool safe = r.guarded && ((int64_t)v[j] > old || (int64_t)v[j] < sinks);
        held[j] = first + 64 * j + lane >= r.len || safe ? PROTECTED : key_of(w[j]);
    }
}

// The slots of a claim that are not victims'.
__device__ __forceinline__ void write_rest(const EvictParams& p, int32_t* out, int len, int64_t free, int64_t v, int64_t first, int64_t step) {
    for (int64_t i = first; i < p.n; i += step) {
        if (i < free) out[i] = (int32_t)(len + i);
        else if (i >= free + v) out[i] = -1;
    }
}

// A row of up to KPT * THREADS slots: wave w holds slots [w * 64 KPT, (w + 1) * 64 KPT).
template <int THREADS, int KPT>
__global__ void __launch_bounds__(THREADS) select_kernel(EvictParams p) {
    constexpr int WAVES = THREADS / 64;
    __shared__ Shared<THREADS> sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Row r = row_of(p, blockIdx.x);
    const int seg = wave * 64 * KPT;
    uint32_t held[KPT];
    {
        // positions stay in registers too, up to 16 a thread; else they are read again (32768 slots of 32 rows, all
        // kept: 36.4 us, spilled; read again: 31.4)
        constexpr int U = KPT < 16 ? KPT : 16;
        const int slot = seg + lane, last = max(r.len - 1, 0);  // (beyond: the last again, no branches)
        int v[U];
        auto positions = [&](int j0) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                v[u] = r.pos[min(slot + 64 * (j0 + u), last)];
            }
        };
        if (r.guarded) positions(0);
#pragma unroll
        for (int j0 = 0; j0 < KPT; j0 += U) {
            float w[U];
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = r.weights[min(slot + 64 * (j0 + u), last)];
#pragma unroll
            for (int u = 0; u < U; ++u) held[j0 + u] = slot + 64 * (j0 + u) < r.len ? key_of(w[u]) : PROTECTED;
        }
        int64_t old = 0x7fffffffll + 1;  // positions above it are protected
        if (p.recent > 0) {
            int top = v[0];
#pragma unroll
            for (int j0 = 0; j0 < KPT; j0 += U) {
                if (j0) positions(j0);
#pragma unroll
                for (int u = 0; u < U; ++u) top = max(top, v[u]);
            }
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) top = max(top, __shfl_xor(top, d));
            if (lane == 0) sh.wave[3][wave] = (uint32_t)top;
            __syncthreads();
            for (int i = 0; i < WAVES; ++i) top = max(top, (int)sh.wave[3][i]);
            old = (int64_t)top - p.recent;
        }
        if (r.guarded) {
#pragma unroll
            for (int j0 = 0; j0 < KPT; j0 += U) {
                if (KPT > U) positions(j0);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if ((int64_t)v[u] > old || (int64_t)v[u] < p.sinks) held[j0 + u] = PROTECTED;
            }
        }
    }
    auto each = [&](auto&& f) {
#pragma unroll
        for (int j = 0; j < KPT; ++j) f(held[j]);
    };

    // candidates, and the range of their keys
    uint32_t low = PROTECTED, high = 0, count = 0;
    each([&](uint32_t k) {
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
    int64_t free;
    const int64_t v = victims(p, r.len, count, free);
    uint32_t edge = 0;
    int64_t ties = 0;
    if (v >= (int64_t)count) {
        if (v > 0) edge = PROTECTED, ties = v - count;
    } else if (v == 1) {  // the lowest needs no search
        edge = low, ties = 1;
    } else if (v > 0) {
        search(sh, each, low, high, (uint32_t)v, lane, wave, edge, ties);
    }

    // ranks: counts of the waves before, then along the wave
    // (asm: or the compiler keeps two masks a key, of the comparisons that it then need not
    // repeat, and spills hundreds of scalar registers)
    uint32_t below = 0, same = 0;
    int at = seg + lane;
    asm("" : "+v"(at));
#pragma unroll
    for (int j = 0; j < KPT; ++j) {
        const bool live = at + 64 * j < r.len;
        below += __popcll(__ballot(live && held[j] < edge));
        same += __popcll(__ballot(live && held[j] == edge));
    }
    if (lane == 0) sh.wave[0][wave] = below, sh.wave[1][wave] = same;
    __syncthreads();
    int64_t gone = 0, seen = 0;
    for (int w = 0; w < wave; ++w) gone += sh.wave[0][w], seen += sh.wave[1][w];
    gone += min(seen, ties);
    int32_t* out = p.out + (int64_t)r.bh * (p.evict ? p.budget : p.n);
    asm("" : "+v"(at), "+v"(edge));
    Writer write{p, out, (uint32_t)free, (uint32_t)ties, (uint32_t)gone, (uint32_t)seen, edge, r.len};
#pragma unroll
    for (int j = 0; j < KPT; ++j) write(held[j], (uint32_t)(at + 64 * j));
    if (!p.evict) write_rest(p, out, r.len, free, v, threadIdx.x, THREADS);
}

// -- rows in parts: blockIdx.x is the row, blockIdx.y the part ---------------
constexpr int PART_THREADS = 256, PART_WAVES = 4, MAX_PARTS = 32;

// f(key, slot) for the part's slots (the ends of rounds past the length among them, as
// PROTECTED); a wave's are consecutive.  Positions above `old` are protected, and below the sinks.
template <class F>
__device__ __forceinline__ void each_of_part(const EvictParams& p, const Row& r, int64_t old, int lane, int wave, F&& f) {
    const int per = p.part / PART_WAVES;
    const int64_t first = (int64_t)blockIdx.y * p.part + wave * per;
    const int rounds = (int)(first >= r.len ? 0 : min((int64_t)per, r.len - first + 63) / 64);
    constexpr int U = 16;  // rounds whose loads are under way together: all of a part of 4096 slots
    for (int j = 0; j < rounds; j += U) {
        int v[U];
        float w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = first + 64 * (j + u) + lane;
            const bool live = i < r.len && j + u < rounds;
            v[u] = r.guarded && live ? r.pos[i] : 0;
            w[u] = live ? r.weights[i] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (j + u >= rounds) break;
            const int64_t i = first + 64 * (j + u) + lane;
            const bool safe = r.guarded && ((int64_t)v[u] > old || (int64_t)v[u] < p.sinks);
            f(i >= r.len || safe ? PROTECTED : key_of(w[u]), i, v[u]);
        }
    }
}

// Range of the keys, protected or not, and the largest position.
__global__ void __launch_bounds__(PART_THREADS) survey_kernel(EvictParams p) {
    __shared__ uint32_t sh[3][PART_WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    EvictParams all = p;
    all.sinks = -0x7fffffffll - 1;  // nothing is protected here
    const Row r = row_of(p, blockIdx.x);
    uint32_t low = PROTECTED, high = 0;
    int top = -0x7fffffff - 1;
    each_of_part(all, r, 0x7fffffffll + 1, lane, wave, [&](uint32_t k, int64_t i, int v) {
        if (i < r.len) low = min(low, k), high = max(high, k), top = max(top, v);
    });
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        low = min(low, (uint32_t)__shfl_xor((int)low, d));
        high = max(high, (uint32_t)__shfl_xor((int)high, d));
        top = max(top, __shfl_xor(top, d));
    }
    if (lane == 0) sh[0][wave] = low, sh[1][wave] = high, sh[2][wave] = (uint32_t)top;
    __syncthreads();
    if (threadIdx.x != 0) return;
    if (blockIdx.y == 0) p.listed[blockIdx.x] = 0;
    for (int w = 0; w < PART_WAVES; ++w) {
        low = min(low, sh[0][w]);
        high = max(high, sh[1][w]);
        top = max(top, (int)sh[2][w]);
    }
    p.survey[(int64_t)blockIdx.x * p.parts + blockIdx.y] = make_int4(top, (int)low, (int)high, 0);
}

struct Range {
    int64_t old;  // positions above it are protected
    uint32_t low, high;
    int shift;    // of the first digit
};

__device__ __forceinline__ Range range_of(const EvictParams& p, int bh, int lane) {
    static_assert(MAX_PARTS <= 64, "a lane takes a part");
    int4 s = make_int4(-0x7fffffff - 1, (int)PROTECTED, 0, 0);
    if (lane < p.parts) s = p.survey[(int64_t)bh * p.parts + lane];
    int top = s.x;
    uint32_t low = (uint32_t)s.y, high = (uint32_t)s.z;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        top = max(top, __shfl_xor(top, d));
        low = min(low, (uint32_t)__shfl_xor((int)low, d));
        high = max(high, (uint32_t)__shfl_xor((int)high, d));
    }
    const int width = high <= low ? 0 : 32 - __clz((int)(high - low));
    return {p.recent > 0 ? (int64_t)top - p.recent : 0x7fffffffll + 1, low, high, width > DIGIT ? width - DIGIT : 0};
}

// The first digit's counts of the part's unprotected keys.
__global__ void __launch_bounds__(PART_THREADS) histogram_kernel(EvictParams p) {
    __shared__ Shared<PART_THREADS> sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Row r = row_of(p, blockIdx.x);
    for (int i = threadIdx.x; i < BINS; i += PART_THREADS) sh.bins[i] = 0;
    const Range g = range_of(p, blockIdx.x, lane);
    __syncthreads();
    each_of_part(p, r, g.old, lane, wave, [&](uint32_t k, int64_t, int) {
        count_key(sh, k != PROTECTED, (k - g.low) >> g.shift, lane);
    });
    __syncthreads();
    uint32_t* hist = p.hist + ((int64_t)blockIdx.x * p.parts + blockIdx.y) * BINS;
    for (int i = threadIdx.x; i < BINS; i += PART_THREADS) hist[i] = sh.bins[i];
}

// The bin of the v-th key, from all parts' counts: {bin, keys before it, keys in it, unprotected keys in all}.
__device__ __forceinline__ uint4 place_of(const EvictParams& p, const Row& r, Shared<PART_THREADS>& sh, int lane, int wave) {
    constexpr int PER = BINS / PART_THREADS;
    const uint32_t* hist = p.hist + (int64_t)r.bh * p.parts * BINS + threadIdx.x * PER;
    uint32_t c[PER] = {};
#pragma unroll 8
    for (int i = 0; i < p.parts; ++i) {
#pragma unroll
        for (int j = 0; j < PER; j += 4) {
            const u32x4 x = *(const u32x4*)(hist + (int64_t)i * BINS + j);
#pragma unroll
            for (int k = 0; k < 4; ++k) c[j + k] += x[k];
        }
    }
    uint32_t count = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) count += c[j];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) count += (uint32_t)__shfl_xor((int)count, d);
    if (lane == 0) sh.wave[0][wave] = count;
    __syncthreads();
    count = 0;
    for (int w = 0; w < PART_WAVES; ++w) count += sh.wave[0][w];
    int64_t free;
    const int64_t v = victims(p, r.len, count, free);
    if (v <= 0 || v >= (int64_t)count) return make_uint4(0, 0, 0, count);
    find_bin(sh, (uint32_t)v, lane, wave, [&](int i) {
        uint32_t x = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) x = (i % PER) == j ? c[j] : x;
        return x;
    });
    return make_uint4(sh.found[0], sh.found[1], sh.found[2], count);
}

// The part's keys in that bin, and its counts.
__global__ void __launch_bounds__(PART_THREADS) collect_kernel(EvictParams p) {
    __shared__ Shared<PART_THREADS> sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Row r = row_of(p, blockIdx.x);
    if (threadIdx.x == 0) sh.listed = 0;
    const uint4 o = place_of(p, r, sh, lane, wave);
    if (blockIdx.y == 0 && threadIdx.x == 0) p.found[blockIdx.x] = o;
    if (o.z == 0) return;  // all unprotected slots go, or none
    const Range g = range_of(p, blockIdx.x, lane);
    const int64_t at = (int64_t)blockIdx.x * p.parts + blockIdx.y;
    uint32_t below = 0;
    // the part's share of the row's list; the order of shares says nothing
    const uint32_t n = p.hist[at * BINS + o.x];
    if (threadIdx.x == 0) sh.list[0] = atomicAdd(&p.listed[blockIdx.x], n);
    __syncthreads();
    const uint32_t start = sh.list[0];
    uint32_t* list = p.list + (int64_t)blockIdx.x * p.parts * p.part + start;
    each_of_part(p, r, g.old, lane, wave, [&](uint32_t k, int64_t, int) {
        const bool in = k != PROTECTED;
        const uint32_t bin = (k - g.low) >> g.shift;
        below += __popcll(__ballot(in && bin < o.x));
        if (in && bin == o.x) list[atomicAdd(&sh.listed, 1u)] = k;
    });
    if (lane == 0) sh.wave[0][wave] = below;
    __syncthreads();
    if (threadIdx.x != 0) return;
    below = 0;
    for (int w = 0; w < PART_WAVES; ++w) below += sh.wave[0][w];
    p.counts[at] = make_int4((int)below, (int)n, (int)start, 0);
}

// The edge, from all parts' lists, and this part's slots.
__global__ void __launch_bounds__(PART_THREADS) choose_kernel(EvictParams p) {
    __shared__ Shared<PART_THREADS> sh;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Row r = row_of(p, blockIdx.x);
    const uint4 o = p.found[blockIdx.x];
    const uint32_t inside = o.z, count = o.w;
    int64_t free;
    const int64_t v = victims(p, r.len, count, free);
    const Range g = range_of(p, blockIdx.x, lane);
    const int64_t row_at = (int64_t)blockIdx.x * p.parts;
    uint32_t edge = 0;
    int64_t ties = 0, gone = 0, seen = 0;
    if (v >= (int64_t)count) {
        if (v > 0) edge = PROTECTED, ties = v - count;
    } else if (v > 0) {
        const uint32_t base = g.low + (o.x << g.shift), rest = (uint32_t)v - o.y;
        int4 n = make_int4(0, 0, 0, 0);  // lane q: the counts of part q
        if (lane < p.parts) n = p.counts[row_at + lane];
        const uint32_t* list = p.list + row_at * p.part;
        if (g.shift == 0) {
            edge = base, ties = rest;
        } else if (inside <= RANKED) {
            if (threadIdx.x < inside) sh.list[threadIdx.x] = list[threadIdx.x];
            __syncthreads();
            rank_listed(sh, inside, rest, edge, ties);
        } else {
            auto each = [&](auto&& f) {
                for (uint32_t i = 64 * wave; i < inside; i += PART_THREADS) f(i + lane < inside ? list[i + lane] : PROTECTED);
            };
            search(sh, each, base, base + min(g.high - base, (1u << g.shift) - 1), rest, lane, wave, edge, ties);
        }
        // of the parts before: keys below the edge, and equal to it
        uint32_t below = wave == 0 && lane < (int)blockIdx.y ? (uint32_t)n.x : 0, same = 0;
        for (uint32_t first = 64 * wave; first < inside; first += PART_THREADS) {
            const uint32_t i = first + lane;
            bool before = false;
            for (int q = 0; q < (int)blockIdx.y; ++q)
                before |= i - (uint32_t)__builtin_amdgcn_readlane(n.z, q) < (uint32_t)__builtin_amdgcn_readlane(n.y, q);
            if (before && i < inside) {
                const uint32_t k = list[i];
                below += k < edge;
                same += k == edge;
            }
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            below += (uint32_t)__shfl_xor((int)below, d);
            same += (uint32_t)__shfl_xor((int)same, d);
        }
        __syncthreads();
        if (lane == 0) sh.wave[0][wave] = below, sh.wave[1][wave] = same;
        __syncthreads();
        for (int w = 0; w < PART_WAVES; ++w) gone += sh.wave[0][w], seen += sh.wave[1][w];
        __syncthreads();
    }
    if (edge == PROTECTED) {
        // every unprotected slot goes, and protected ones by slot: the parts before hold their slots' share
        const int64_t first = (int64_t)blockIdx.y * p.part;
        const int64_t slots = min(first, (int64_t)r.len);
        int64_t loose = 0;
        const uint32_t* hist = p.hist + row_at * BINS;
        uint32_t n = 0;
        for (int q = 0; q < (int)blockIdx.y; ++q)
            for (int i = threadIdx.x; i < BINS; i += PART_THREADS) n += hist[(int64_t)q * BINS + i];
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) n += (uint32_t)__shfl_xor((int)n, d);
        if (lane == 0) sh.wave[0][wave] = n;
        __syncthreads();
        for (int w = 0; w < PART_WAVES; ++w) loose += sh.wave[0][w];
        __syncthreads();
        gone = loose, seen = slots - loose;
    }
    // this part's waves; the keys of a part of 4096 slots stay in registers
    constexpr int HELD = 16;
    const bool hold = p.part == HELD * PART_THREADS;
    const int64_t first = (int64_t)blockIdx.y * p.part + wave * (p.part / PART_WAVES);
    uint32_t held[HELD];
    uint32_t below = 0, same = 0;
    auto count_slot = [&](uint32_t k, int64_t i) {
        const bool live = i < r.len;
        below += __popcll(__ballot(live && k < edge));
        same += __popcll(__ballot(live && k == edge));
    };
    if (hold) {
        hold_keys<HELD>(r, first, g.old, p.sinks, lane, held);
#pragma unroll
        for (int j = 0; j < HELD; ++j) count_slot(held[j], first + 64 * j + lane);
    } else {
        each_of_part(p, r, g.old, lane, wave, [&](uint32_t k, int64_t i, int) { count_slot(k, i); });
    }
    if (lane == 0) sh.wave[0][wave] = below, sh.wave[1][wave] = same;
    __syncthreads();
    for (int w = 0; w < wave; ++w) gone += sh.wave[0][w], seen += sh.wave[1][w];
    gone += min(seen, ties);
    int32_t* out = p.out + (int64_t)r.bh * (p.evict ? p.budget : p.n);
    Writer write{p, out, (uint32_t)free, (uint32_t)ties, (uint32_t)gone, (uint32_t)seen, edge, r.len};
    if (hold) {
#pragma unroll
        for (int j = 0; j < HELD; ++j) write(held[j], (uint32_t)(first + 64 * j + lane));
    } else {
        each_of_part(p, r, g.old, lane, wave, [&](uint32_t k, int64_t i, int) { write(k, (uint32_t)i); });
    }
    if (!p.evict) write_rest(p, out, r.len, free, v, (int64_t)blockIdx.y * PART_THREADS + threadIdx.x, (int64_t)p.parts * PART_THREADS);
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

constexpr int64_t WHOLE_ROW = 32768;  // slots that one workgroup chooses among

// Parts of a row, and the workspace: 4096 slots a part, up to 32 parts of more.
struct Plan {
    int parts = 0, part = 0;
    uint64_t kept = 0, survey = 0, hist = 0, found = 0, listed = 0, counts = 0, list = 0, bytes = 0;
};

Plan make_plan(const rsfa_cache4_evict_args* a, bool evict) {
    Plan p;
    const int64_t bh = a->cache.z * a->cache.h, c = a->cache.capacity;
    auto take = [&](uint64_t n) {
        const uint64_t here = p.bytes;
        p.bytes += (n + 255) / 256 * 256;
        return here;
    };
    if (evict) p.kept = take((uint64_t)bh * a->budget * 4);
    if (c > WHOLE_ROW) {
        p.parts = (int)std::min<int64_t>(MAX_PARTS, (c + 4095) / 4096);
        p.part = (int)(((c + p.parts - 1) / p.parts + 255) / 256 * 256);
        const uint64_t all = (uint64_t)bh * p.parts;
        p.survey = take(all * sizeof(int4));
        p.hist = take(all * BINS * 4);
        p.found = take((uint64_t)bh * sizeof(uint4));
        p.listed = take((uint64_t)bh * 4);
        p.counts = take(all * sizeof(int4));
        p.list = take(all * p.part * 4);
    }
    return p;
}

int check_evict(const rsfa_cache4_evict_args* a, bool evict) {
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
    return RSFA_OK;
}

int evict_launch(const rsfa_cache4_evict_args* a, bool evict, void* stream) {
    const int st = check_evict(a, evict);
    if (st != RSFA_OK) return st;
    if (!evict && !a->out) return RSFA_E_NULL;
    if (((uintptr_t)a->lengths | (uintptr_t)a->out) & 3) return RSFA_E_ALIGN;
    const Plan plan = make_plan(a, evict);
    if (plan.bytes) {
        if (!a->workspace || a->workspace_bytes < plan.bytes) return RSFA_E_WORKSPACE;
        if ((uintptr_t)a->workspace & 15) return RSFA_E_ALIGN;
    }
    const int64_t bh = a->cache.z * a->cache.h;
    EvictParams p{};
    p.c = a->cache;
    if (evict) p.into = a->into;
    p.lengths = a->lengths, p.length = a->length;
    p.n = a->n, p.budget = a->budget, p.recent = a->recent, p.sinks = a->sinks;
    p.evict = evict ? 1 : 0;
    char* ws = (char*)a->workspace;
    p.out = evict ? (int32_t*)(ws + plan.kept) : a->out;
    p.parts = plan.parts, p.part = plan.part;
    if (plan.parts) {
        p.survey = (int4*)(ws + plan.survey);
        p.hist = (uint32_t*)(ws + plan.hist);
        p.found = (uint4*)(ws + plan.found);
        p.listed = (uint32_t*)(ws + plan.listed);
        p.counts = (int4*)(ws + plan.counts);
        p.list = (uint32_t*)(ws + plan.list);
    }
    const int64_t blocks = evict ? (bh * a->budget * (a->cache.head_dim / 32) + 255) / 256 : 1;
    if (blocks > 0x7fffffff) return RSFA_E_CACHE;
    void* args[] = {&p};
    auto launch = [&](const void* fn, dim3 grid, int threads) {
        return hipLaunchKernel(fn, grid, dim3((unsigned)threads), args, 0, (hipStream_t)stream) == hipSuccess;
    };
    if (!plan.parts) {
        // eight slots a thread (4096 slots of 64 rows, with the copy: 13.8 us, 15.9 with 16), until that takes
        // more than the largest workgroup
        const int64_t c = a->cache.capacity;
        const void* fn = (const void*)&select_kernel<1024, 8>;
        int threads = 1024;
        if (c <= 2048) fn = (const void*)&select_kernel<256, 8>, threads = 256;
        else if (c <= 4096) fn = (const void*)&select_kernel<512, 8>, threads = 512;
        else if (c > 16384) fn = (const void*)&select_kernel<1024, 32>;
        else if (c > 8192) fn = (const void*)&select_kernel<1024, 16>;
        if (!launch(fn, dim3((unsigned)bh), threads)) return RSFA_E_LAUNCH;
    } else {
        const dim3 grid((unsigned)bh, (unsigned)plan.parts);
        if (!launch((const void*)&survey_kernel, grid, PART_THREADS) || !launch((const void*)&histogram_kernel, grid, PART_THREADS) ||
            !launch((const void*)&collect_kernel, grid, PART_THREADS) || !launch((const void*)&choose_kernel, grid, PART_THREADS))
            return RSFA_E_LAUNCH;
    }
    if (!evict) return RSFA_OK;
    const int64_t d = a->cache.head_dim;
    const void* fn = d == 32    ? (const void*)&gather_kernel<32>
                     : d == 64  ? (const void*)&gather_kernel<64>
                     : d == 128 ? (const void*)&gather_kernel<128>
                                : (const void*)&gather_kernel<256>;
    return launch(fn, dim3((unsigned)blocks), 256) ? RSFA_OK : RSFA_E_LAUNCH;
}

}  // namespace

extern "C" {

uint64_t rsfa_cache4_evict_workspace_bytes(const rsfa_cache4_evict_args* a, int32_t evict) {
    return check_evict(a, evict != 0) == RSFA_OK ? make_plan(a, evict != 0).bytes : 0;
}

int rsfa_cache4_claim(const rsfa_cache4_evict_args* a, void* stream) { return evict_launch(a, false, stream); }
int rsfa_cache4_evict(const rsfa_cache4_evict_args* a, void* stream) { return evict_launch(a, true, stream); }

}  // extern "C"
