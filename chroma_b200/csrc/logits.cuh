// What is done to logits before a token is chosen from them: penalties for tokens that occurred, biases, temperature,
// the mask of a grammar, and the greedy choice.
//
// Few rows (k_logits): one CTA takes a segment of one row, counts the row's history into a table of its segment in shared
// memory, adds the biases of its segment in list order, and passes over the logits once, 16 bytes a thread. Many rows: reading
// the history once for every segment would cost more than the logits, so k_logits_heard finishes the entries that
// occurred or have a bias, through a hash table, and leaves their bits; k_logits_rest streams the others. The best of each
// segment is left for a last, small launch. No table of counts is kept between calls. The arithmetic is rounded operation by
// operation (no fused multiply-add), so that results do not depend on how the compiler groups it, and equal logits stay equal.
//
// Bound: one row by the latency of a few dependent reads (history of 500: 9 us one call after another, as long as the
// host's call). 64 rows of 201,088 with histories of 50-4,096, 50 biases and a mask, fp32: 32 us, 3.2 TB/s, where the bytes
// alone take 16: 8 us are the chain of row length, history, table, logits of the first launch, under which only the first
// segments of the second are read (its stores wait, which a call in place needs and another would not), and the second one
// issues 20 instructions an entry (five of them the division by the temperature); 128 rows 55 us. All in one launch, with segments of 4,096 to 16,384 entries on 128 to 1,024 threads, took 45 to 57 us for
// the 64 rows; a table with a place for each of 16,384 entries in place of the hash table 47.
#pragma once

#include <limits.h>

#include <type_traits>

#include "paged.cuh"

namespace cb200 {

// Entries of a segment: 4 or 16 a thread. Few rows are cut finer, so that they reach all SMs. (Rows of 201,088, all in one
// launch with 1,024 entries a segment and in two with 4,096: one 12 and 14 us, two 14 and 16, four 16 and 16, six 18 and 18,
// twelve 25 and 18, sixty-four 80 and 33, by events around a graph.)
constexpr int kLogitsThreads = 256, kLogitsShort = 4 * kLogitsThreads, kLogitsLong = 16 * kLogitsThreads;
// A token's word in the table of its segment: it occurs in the prompt, it has a bias, and how often it occurs after that.
constexpr unsigned kHeardBit = 0x80000000u, kBiasBit = 0x40000000u, kTimes = 0x3fffffffu;
constexpr int kLogitsListed = 256;  // biases of a segment that are kept in shared memory; more are read again from the list

struct LogitsArgs {
    const void* logits;
    void* out;
    const int *history, *lengths, *prompts;
    const float *repetition, *presence, *frequency, *temperature;
    const int* bias_ids;
    const float* bias;
    const unsigned* mask;
    unsigned long long* best;  // [rows][segments] argmax keys, or nullptr
    int64_t stride, out_stride, history_stride, bias_ids_stride, bias_stride, mask_stride;
    unsigned* special;         // [rows][special_stride] bits: entries that occurred or have a bias; or nullptr
    int special_stride, best_at;  // best_at: this launch's first segment of `best`
    FastDiv by_ctas;              // d: CTAs that share a row's words of 32 entries, in turn
    int vocab, width, biases, segments;
    int vector, history_vector;  // rows of logits and out, of the history, are 16-byte aligned
};

// a / b with b's correctly rounded reciprocal y, correctly rounded: a quotient within a unit in the last place, and the
// remainder that it leaves, exact by fused multiply-add (Markstein, "Computation of elementary functions on the IBM RISC
// System/6000 processor", IBM J. Res. Dev. 34, 1990). For a and b far from the ends of the exponent's range. A row has one
// divisor, so this takes five instructions where a division takes a branch and two to three times as many.
__device__ __forceinline__ float divided(float a, float b, float y) {
    float q = __fmul_rn(a, y);
    q = __fmaf_rn(__fmaf_rn(-q, b, a), y, q);
    return __fmaf_rn(__fmaf_rn(-q, b, a), y, q);
}

__device__ __noinline__ float divided_anyhow(float a, float b) { return __fdiv_rn(a, b); }

// The sum of the biases of token `begin` + i, in the order of the row's list. `listed` of the list lie in the segment that
// begins there; as many as there is room for are in shared memory, in any order, with their places in the list.
__device__ __noinline__ float bias_sum(const int* all_ids, const float* all, int biases, int token, int i, int listed, const int* ids,
                                       const int* places, const float* values) {
    float sum = 0.f;
    if (listed > kLogitsListed) {
        for (int j = 0; j < biases; ++j)
            if (all_ids[j] == token) sum = __fadd_rn(sum, all[j]);
        return sum;
    }
    for (int last = -1;;) {
        int next = INT_MAX, which = 0;
        for (int j = 0; j < listed; ++j)
            if (ids[j] == i && places[j] > last && places[j] < next) next = places[which = j];
        if (next == INT_MAX) return sum;
        sum = __fadd_rn(sum, values[which]);
        last = next;
    }
}

template <typename T> __global__ void __launch_bounds__(kLogitsThreads, 5) k_logits(LogitsArgs a) {
    constexpr int kPer = 16 / sizeof(T), kSegment = kLogitsShort;
    __shared__ __align__(16) unsigned counts[kSegment];
    __shared__ unsigned special[kSegment / 32];  // entries that occurred or have a bias: they are left to the second pass
    __shared__ uint16_t specials[kSegment];
    __shared__ int listed_ids[kLogitsListed], listed_at[kLogitsListed];
    __shared__ float listed[kLogitsListed];
    __shared__ int s_listed, s_specials;
    __shared__ unsigned long long keys[kLogitsThreads / 32];
    asm volatile("griddepcontrol.launch_dependents;" :::);
    const int row = blockIdx.y, begin = blockIdx.x * kSegment, n = min(kSegment, a.vocab - begin);
    const float temp = a.temperature ? a.temperature[row] : 0.f;
    const bool heard = a.history, biased = a.bias_ids, tabled = heard || biased;
    const T* in = static_cast<const T*>(a.logits) + row * a.stride + begin;
    T* out = static_cast<T*>(a.out) + row * a.out_stride + begin;
    const unsigned* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    // The first of the history and of the biases, and this thread's words: all under way at once.
    constexpr int kEarly = 2;
    const int len = heard ? min(max(a.lengths[row], 0), a.width) : 0, prompt = heard && a.prompts ? a.prompts[row] : 0;
    const int* history = a.history + row * a.history_stride;
    const auto tokens = [&](int i) {  // entries i .. i + 3
        if (a.history_vector && i + 4 <= a.width) return __ldg(reinterpret_cast<const int4*>(history + i));
        return make_int4(i < a.width ? __ldg(history + i) : -1, i + 1 < a.width ? __ldg(history + i + 1) : -1,
                         i + 2 < a.width ? __ldg(history + i + 2) : -1, i + 3 < a.width ? __ldg(history + i + 3) : -1);
    };
    int4 early[kEarly];
#pragma unroll
    for (int v = 0; v < kEarly; ++v)
        if (heard) early[v] = tokens(4 * (threadIdx.x + v * kLogitsThreads));
    int early_id = -1;
    if (biased && int(threadIdx.x) < a.biases) early_id = __ldg(a.bias_ids + row * a.bias_ids_stride + threadIdx.x);
    constexpr int kWords = (kSegment + kPer * kLogitsThreads - 1) / (kPer * kLogitsThreads);
    uint4 words[kWords];
    unsigned allowed[kWords];
#pragma unroll
    for (int v = 0; v < kWords; ++v) {
        const int i = kPer * (threadIdx.x + v * kLogitsThreads);
        if (!a.vector || i + kPer > n) continue;
        words[v] = *reinterpret_cast<const uint4*>(in + i);
        allowed[v] = mask ? __ldg(mask + ((begin + i) >> 5)) >> ((begin + i) & 31) : ~0u;
    }
    if (tabled) {
        for (int i = 4 * threadIdx.x; i < kSegment; i += 4 * kLogitsThreads) *reinterpret_cast<uint4*>(counts + i) = make_uint4(0, 0, 0, 0);
        for (int i = threadIdx.x; i < kSegment / 32; i += kLogitsThreads) special[i] = 0;
        if (threadIdx.x == 0) s_listed = s_specials = 0;
        __syncthreads();
        const auto mark = [&](unsigned t, unsigned before) {  // the first who touches an entry puts it on the list
            if (before) return;
            specials[atomicAdd(&s_specials, 1)] = uint16_t(t);
            atomicOr(&special[t >> 5], 1u << (t & 31));
        };
        const auto hear = [&](int i, int token) {
            const unsigned t = unsigned(token - begin);
            if (i < len && t < unsigned(n)) mark(t, i < prompt ? atomicOr(&counts[t], kHeardBit) : atomicAdd(&counts[t], 1u));
        };
        const auto hear4 = [&](int i, const int4& x) {
            hear(i, x.x);
            hear(i + 1, x.y);
            hear(i + 2, x.z);
            hear(i + 3, x.w);
        };
        if (heard) {
#pragma unroll
            for (int v = 0; v < kEarly; ++v) hear4(4 * (threadIdx.x + v * kLogitsThreads), early[v]);
#pragma unroll 2
            for (int i = 4 * (threadIdx.x + kEarly * kLogitsThreads); i < len; i += 4 * kLogitsThreads) hear4(i, tokens(i));
        }
        if (biased)
            for (int i = threadIdx.x; i < a.biases; i += kLogitsThreads) {
                const unsigned t = unsigned((i < kLogitsThreads ? early_id : __ldg(a.bias_ids + row * a.bias_ids_stride + i)) - begin);
                if (t >= unsigned(n)) continue;
                mark(t, atomicOr(&counts[t], kBiasBit));
                const int at = atomicAdd(&s_listed, 1);
                if (at < kLogitsListed) {
                    listed_ids[at] = int(t);
                    listed_at[at] = i;
                    listed[at] = a.bias[row * a.bias_stride + i];
                }
            }
        __syncthreads();
    }
    const bool usual_temp = fabsf(temp) > 0x1p-30f && fabsf(temp) < 0x1p30f;
    const float per_temp = __frcp_rn(temp);
    float top = -INFINITY;  // of this thread's entries, and where: the first of equals, the first NaN before all
    int where = -1;
    const auto choose = [&](float x, int i) {
        if (!(x <= top) && top == top) {
            top = x;
            where = i;
        }
    };
    const auto finished = [&](float x, unsigned on) {
        if (temp != 0.f) x = divided_anyhow(x, temp);
        return on ? Store<T>::round(x) : -INFINITY;
    };
    const auto allowed_at = [&](int i) { return mask ? __ldg(mask + ((begin + i) >> 5)) >> ((begin + i) & 31) & 1 : 1u; };
    const auto special_at = [&](int i) { return tabled && (special[i >> 5] >> (i & 31) & 1); };
    const auto one = [&](int i) {
        if (special_at(i)) return;
        const float x = finished(Store<T>::load(in + i), allowed_at(i));
        choose(x, i);
        Store<T>::store(out + i, x);
    };
    if (a.vector) {
        const int first = kPer * threadIdx.x;
        if (first < n) where = first;
#pragma unroll
        for (int v = 0; v < kWords; ++v) {
            const int i = kPer * (threadIdx.x + v * kLogitsThreads);
            if (i + kPer > n) {
                for (int e = i; e < n; ++e) one(e);
                continue;
            }
            const unsigned left = tabled ? special[i >> 5] >> (i & 31) & ((1u << kPer) - 1) : 0u, on = allowed[v] & ~left;
            alignas(16) T raw[kPer];
            *reinterpret_cast<uint4*>(raw) = words[v];
            float x[kPer];
#pragma unroll
            for (int e = 0; e < kPer; ++e) x[e] = Store<T>::load(raw + e);
            if (temp != 0.f) {
                bool usual = usual_temp;
#pragma unroll
                for (int e = 0; e < kPer; ++e) usual = usual && fabsf(x[e]) > 0x1p-60f && fabsf(x[e]) < 0x1p60f;
                if (usual)
#pragma unroll
                    for (int e = 0; e < kPer; ++e) x[e] = divided(x[e], temp, per_temp);
                else
#pragma unroll
                    for (int e = 0; e < kPer; ++e) x[e] = divided_anyhow(x[e], temp);
            }
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                x[e] = on >> e & 1 ? Store<T>::round(x[e]) : -INFINITY;
                choose(x[e], i + e);
                Store<T>::store(raw + e, x[e]);
            }
            if (!left) *reinterpret_cast<uint4*>(out + i) = *reinterpret_cast<const uint4*>(raw);
            else
#pragma unroll
                for (int e = 0; e < kPer; ++e)
                    if (!(left >> e & 1)) out[i + e] = raw[e];
        }
    } else {
        if (int(threadIdx.x) < n) where = threadIdx.x;
        for (int i = threadIdx.x; i < n; i += kLogitsThreads) one(i);
    }
    if (tabled && s_specials) {
        // The entries that occurred or have a bias, dealt out anew: most of them crowd into few segments, and few words.
        const float r = a.repetition ? a.repetition[row] : 1.f, f = a.frequency ? a.frequency[row] : 0.f;
        const float pr = a.presence ? a.presence[row] : 0.f;
        for (int k = threadIdx.x; k < s_specials; k += kLogitsThreads) {
            const int i = specials[k];
            const unsigned c = counts[i], times = c & kTimes;
            float x = Store<T>::load(in + i);
            if (c & ~kBiasBit) {
                x = x > 0.f ? divided_anyhow(x, r) : __fmul_rn(x, r);
                if (times) x = __fsub_rn(__fsub_rn(x, __fmul_rn(f, float(times))), pr);
            }
            if (c & kBiasBit) x = __fadd_rn(x, bias_sum(a.bias_ids + row * a.bias_ids_stride, a.bias + row * a.bias_stride, a.biases, begin + i, i, s_listed, listed_ids, listed_at, listed));
            x = finished(x, allowed_at(i));
            Store<T>::store(out + i, x);
            // Not in ascending order: of equals the lower index.
            if (x == top && where >= 0 ? i < where : !(x <= top) && top == top) {
                top = x;
                where = i;
            } else if (x != x && top != top && i < where) where = i;
        }
    }
    if (!a.best) return;
    unsigned long long best = where < 0 ? 0 : argmax_key(top + 0.0f, begin + where);  // + 0: a negative zero equals a positive one
    for (int o = 16; o; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
    }
    if ((threadIdx.x & 31) == 0) keys[threadIdx.x >> 5] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kLogitsThreads / 32; ++w) best = keys[w] > best ? keys[w] : best;
        a.best[int64_t(row) * a.segments + blockIdx.x] = best;
    }
}

// Entries of many rows that occurred or have a bias. A row's words of 32 entries are dealt out to `by_ctas.d` CTAs, so that the
// low ids, which occur most, meet all of them. Each CTA counts its share of the history in a hash table that has room for every
// entry that can come (at least a quarter stays empty), finishes those entries, and leaves bits of where they are.
constexpr int kHeardThreads = 1024, kHeardSlots = 8192, kHeardMost = 6144, kHeardWords = 8192;
struct HeardTable {
    int ids[kHeardSlots];
    unsigned counts[kHeardSlots];
    uint16_t used[kHeardMost];
    int listed_ids[kLogitsListed], listed_at[kLogitsListed];
    float listed[kLogitsListed];
    unsigned long long keys[kHeardThreads / 32];
    int n_listed, n_used;
    unsigned special[];  // words of the CTA
};

template <typename T> __global__ void __launch_bounds__(kHeardThreads, 1) k_logits_heard(LogitsArgs a) {
    extern __shared__ __align__(16) uint8_t heard_smem[];
    HeardTable& sm = *reinterpret_cast<HeardTable*>(heard_smem);
    asm volatile("griddepcontrol.launch_dependents;" :::);
    const int row = blockIdx.y, ctas = a.by_ctas.d, words = (a.special_stride + ctas - 1) / ctas;
    const T* in = static_cast<const T*>(a.logits) + row * a.stride;
    T* out = static_cast<T*>(a.out) + row * a.out_stride;
    const int* history = a.history + row * a.history_stride;
    const int* bias_ids = a.bias_ids + row * a.bias_ids_stride;
    const float* bias = a.bias + row * a.bias_stride;
    const auto tokens = [&](int i) {  // entries i .. i + 3
        if (a.history_vector && i + 4 <= a.width) return __ldg(reinterpret_cast<const int4*>(history + i));
        return make_int4(i < a.width ? __ldg(history + i) : -1, i + 1 < a.width ? __ldg(history + i + 1) : -1,
                         i + 2 < a.width ? __ldg(history + i + 2) : -1, i + 3 < a.width ? __ldg(history + i + 3) : -1);
    };
    int4 next = make_int4(-1, -1, -1, -1);
    if (a.history) next = tokens(4 * threadIdx.x);
    const int len = a.history ? min(max(a.lengths[row], 0), a.width) : 0, prompt = a.history && a.prompts ? a.prompts[row] : 0;
    for (int i = 4 * threadIdx.x; i < kHeardSlots; i += 4 * kHeardThreads) {
        *reinterpret_cast<int4*>(sm.ids + i) = make_int4(-1, -1, -1, -1);
        *reinterpret_cast<uint4*>(sm.counts + i) = make_uint4(0, 0, 0, 0);
    }
    for (int i = threadIdx.x; i < words; i += kHeardThreads) sm.special[i] = 0;
    if (threadIdx.x == 0) sm.n_listed = sm.n_used = 0;
    __syncthreads();
    // The slot of an entry of this CTA, -1 for others.
    const auto slot = [&](int token) {
        if (unsigned(token) >= unsigned(a.vocab)) return -1;
        const unsigned word = unsigned(token) >> 5, at = a.by_ctas.div(word);
        if (word - at * ctas != blockIdx.x) return -1;
        unsigned h = unsigned(token) * 2654435761u >> 19;  // 13 bits of the golden ratio's multiple
        while (true) {
            int id = *reinterpret_cast<volatile int*>(sm.ids + h);
            if (id == -1) {
                id = atomicCAS(sm.ids + h, -1, token);
                if (id == -1) {
                    sm.used[atomicAdd(&sm.n_used, 1)] = uint16_t(h);
                    atomicOr(&sm.special[at], 1u << (token & 31));
                    return int(h);
                }
            }
            if (id == token) return int(h);
            h = (h + 1) % kHeardSlots;
        }
    };
    const auto hear = [&](int i, int token) {
        const int h = i < len ? slot(token) : -1;
        if (h >= 0) {
            if (i < prompt) atomicOr(&sm.counts[h], kHeardBit);
            else atomicAdd(&sm.counts[h], 1u);
        }
    };
    for (int i = 4 * threadIdx.x; i < len; i += 4 * kHeardThreads) {
        const int4 x = next;
        if (i + 4 * kHeardThreads < len) next = tokens(i + 4 * kHeardThreads);
        hear(i, x.x);
        hear(i + 1, x.y);
        hear(i + 2, x.z);
        hear(i + 3, x.w);
    }
    if (a.bias_ids)
        for (int i = threadIdx.x; i < a.biases; i += kHeardThreads) {
            const int h = slot(__ldg(bias_ids + i));
            if (h < 0) continue;
            atomicOr(&sm.counts[h], kBiasBit);
            const int at = atomicAdd(&sm.n_listed, 1);
            if (at < kLogitsListed) {
                sm.listed_ids[at] = h;
                sm.listed_at[at] = i;
                sm.listed[at] = bias[i];
            }
        }
    __syncthreads();
    for (int i = threadIdx.x, word; i < words && (word = i * ctas + blockIdx.x) < a.special_stride; i += kHeardThreads)
        a.special[int64_t(row) * a.special_stride + word] = sm.special[i];
    const float temp = a.temperature ? a.temperature[row] : 0.f, r = a.repetition ? a.repetition[row] : 1.f;
    const float f = a.frequency ? a.frequency[row] : 0.f, pr = a.presence ? a.presence[row] : 0.f;
    unsigned long long best = 0;
    for (int k = threadIdx.x; k < sm.n_used; k += kHeardThreads) {
        const int h = sm.used[k], i = sm.ids[h];
        const unsigned c = sm.counts[h], times = c & kTimes;
        const unsigned on = a.mask ? __ldg(a.mask + row * a.mask_stride + (i >> 5)) >> (i & 31) & 1 : 1u;
        float x = Store<T>::load(in + i);
        if (c & ~kBiasBit) {
            x = x > 0.f ? divided_anyhow(x, r) : __fmul_rn(x, r);
            if (times) x = __fsub_rn(__fsub_rn(x, __fmul_rn(f, float(times))), pr);
        }
        if (c & kBiasBit) x = __fadd_rn(x, bias_sum(bias_ids, bias, a.biases, i, h, sm.n_listed, sm.listed_ids, sm.listed_at, sm.listed));
        if (temp != 0.f) x = divided_anyhow(x, temp);
        x = on ? Store<T>::round(x) : -INFINITY;
        Store<T>::store(out + i, x);
        const unsigned long long key = argmax_key(x + 0.0f, i);  // + 0: a negative zero equals a positive one
        best = key > best ? key : best;
    }
    if (!a.best) return;
    for (int o = 16; o; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
    }
    if ((threadIdx.x & 31) == 0) sm.keys[threadIdx.x >> 5] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kHeardThreads / 32; ++w) best = sm.keys[w] > best ? sm.keys[w] : best;
        a.best[int64_t(row) * a.segments + a.best_at + blockIdx.x] = best;
    }
}

// The largest of three, or NaN if one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float m;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}

// The entries of many rows that neither occurred nor have a bias, while the launch before still finds out which did (what
// is read of the others before its end is not used). 16 entries a thread stay in registers until the segment's largest
// is known; only then the few threads that hold it look where.
template <typename T> __global__ void __launch_bounds__(kLogitsThreads, 5) k_logits_rest(LogitsArgs a) {
    constexpr int kPer = 16 / sizeof(T), kWords = kLogitsLong / (kPer * kLogitsThreads);
    __shared__ __align__(16) unsigned tops[kLogitsThreads / 32];
    __shared__ int s_where;
    asm volatile("griddepcontrol.launch_dependents;" :::);
    const int row = blockIdx.y, begin = blockIdx.x * kLogitsLong, n = min(kLogitsLong, a.vocab - begin);
    const T* in = static_cast<const T*>(a.logits) + row * a.stride + begin;
    T* out = static_cast<T*>(a.out) + row * a.out_stride + begin;
    const float temp = a.temperature ? a.temperature[row] : 0.f;
    const bool usual_temp = fabsf(temp) > 0x1p-30f && fabsf(temp) < 0x1p30f;
    const float per_temp = __frcp_rn(temp);
    constexpr unsigned kAll = (1u << kPer) - 1;
    const int at = kPer * threadIdx.x, shift = at & 31;  // the same bits of a word in every vector
    float x[kWords][kPer], top = -INFINITY;
    const auto pass = [&](auto whole) {  // whole: every vector of 16 bytes lies in the row, and is aligned
        constexpr bool kWhole = decltype(whole)::value;
        alignas(16) T raw[kWords][kPer];
        unsigned on[kWords], left[kWords];
        const T* from = in + at;
        const unsigned* mask = a.mask + row * a.mask_stride + ((begin + at) >> 5);
#pragma unroll
        for (int v = 0; v < kWords; ++v) {
            constexpr int kStep = kPer * kLogitsThreads;
            if (kWhole) *reinterpret_cast<uint4*>(raw[v]) = *reinterpret_cast<const uint4*>(from + v * kStep);
            else
#pragma unroll
                for (int e = 0; e < kPer; ++e) raw[v][e] = at + v * kStep + e < n ? from[v * kStep + e] : T(0.f);
            on[v] = a.mask && (kWhole || at + v * kStep < n) ? __ldg(mask + v * (kStep / 32)) : ~0u;
            left[v] = 0;
        }
        if (a.special) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            const unsigned* special = a.special + int64_t(row) * a.special_stride + ((begin + at) >> 5);
#pragma unroll
            for (int v = 0; v < kWords; ++v)
                if (kWhole || at + v * kPer * kLogitsThreads < n) left[v] = __ldcg(special + v * (kPer * kLogitsThreads / 32));
        }
        float low = INFINITY, high = 0.f;
#pragma unroll
        for (int v = 0; v < kWords; ++v)
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                x[v][e] = Store<T>::load(raw[v] + e);
                if (kWhole || at + v * kPer * kLogitsThreads + e < n) {
                    low = fminf(low, fabsf(x[v][e]));
                    high = fmaxf(high, fabsf(x[v][e]));
                }
            }
        if (temp != 0.f) {
            if (usual_temp && low > 0x1p-60f && high < 0x1p60f)
#pragma unroll
                for (int v = 0; v < kWords; ++v)
#pragma unroll
                    for (int e = 0; e < kPer; ++e) x[v][e] = divided(x[v][e], temp, per_temp);
            else
#pragma unroll
                for (int v = 0; v < kWords; ++v)
#pragma unroll
                    for (int e = 0; e < kPer; ++e) x[v][e] = divided_anyhow(x[v][e], temp);
        }
        T* to = out + at;
#pragma unroll
        for (int v = 0; v < kWords; ++v) {
            const int i = at + v * kPer * kLogitsThreads;
            unsigned skip = left[v] >> shift & kAll;
            if (!kWhole && i + kPer > n) skip |= i < n ? kAll << (n - i) & kAll : kAll;
            const unsigned open = on[v] >> shift & ~skip;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                x[v][e] = open & (1u << e) ? Store<T>::round(x[v][e]) : -INFINITY;
                Store<T>::store(raw[v] + e, x[v][e]);
            }
#pragma unroll
            for (int e = 0; e < kPer; e += 2) top = max3_nan(top, x[v][e], x[v][e + 1]);
            if (kWhole && !skip) *reinterpret_cast<uint4*>(to + v * kPer * kLogitsThreads) = *reinterpret_cast<const uint4*>(raw[v]);
            else
#pragma unroll
                for (int e = 0; e < kPer; ++e)
                    if (!(skip & (1u << e))) to[v * kPer * kLogitsThreads + e] = raw[v][e];
        }
    };
    if (threadIdx.x == 0) s_where = INT_MAX;
    if (a.vector && n == kLogitsLong) pass(std::true_type());
    else pass(std::false_type());
    if (!a.best) return;
    const unsigned key = unsigned(argmax_key(top + 0.0f, 0) >> 32);  // + 0: a negative zero equals a positive one
    const unsigned warp_key = __reduce_max_sync(0xffffffffu, key);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = warp_key;
    __syncthreads();
    unsigned best = 0;
#pragma unroll
    for (int w = 0; w < kLogitsThreads / 32; ++w) best = max(best, tops[w]);
    if (key == best) {
        int where = INT_MAX;
#pragma unroll
        for (int v = kWords - 1; v >= 0; --v)
#pragma unroll
            for (int e = kPer - 1; e >= 0; --e)
                if (x[v][e] == top || (x[v][e] != x[v][e] && top != top)) where = kPer * (threadIdx.x + v * kLogitsThreads) + e;
        atomicMin(&s_where, where);
    }
    __syncthreads();
    if (threadIdx.x == 0)
        a.best[int64_t(row) * a.segments + blockIdx.x] =
            (static_cast<unsigned long long>(best) << 32) | (0xffffffffu - static_cast<unsigned>(begin + s_where));
}

// The best of a row's segments; one warp per row.
[[maybe_unused]] static __global__ void __launch_bounds__(32) k_logits_pick(const unsigned long long* best, int segments,
                                                                           int64_t* argmax) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    unsigned long long top = 0;
    for (int i = threadIdx.x; i < segments; i += 32) {
        const unsigned long long key = best[int64_t(blockIdx.x) * segments + i];
        top = key > top ? key : top;
    }
    for (int o = 16; o; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, top, o);
        top = other > top ? other : top;
    }
    if (threadIdx.x == 0) argmax[blockIdx.x] = argmax_index(top);
}

}  // namespace cb200
