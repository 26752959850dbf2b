// What is done to logits before a token is chosen from them: penalties for tokens that occurred, biases, temperature,
// the mask of a grammar, and the greedy choice.
//
// One CTA takes a segment of one row: it counts the row's history into a table of its segment in shared memory, adds the
// biases of its segment in list order, and passes over the logits once, 16 bytes a thread at a time. No table of counts is
// kept between calls. The arithmetic is rounded operation by operation (no fused multiply-add), so that results do not
// depend on how the compiler groups it, and equal logits stay equal. The best of each segment is left for a second, small
// launch.
//
// Bound by latency: each CTA's chain of row length, history, table, logits, best of the segment is longer than its
// share of the stream. 64 rows of 201,088 with histories of 50-4,096, 50 biases and a mask, fp32: 47 us, 2.2 TB/s (the
// bytes alone take 16); one row with a history of 500: 9 us one call after another. Segments of 4,096 to 16,384
// entries on 128 to 1,024 threads, with one to four words of history under way before the table is cleared, all took
// 45 to 57 us for the 64 rows.
#pragma once

#include <limits.h>

#include "common.cuh"

namespace cb200 {

// Entries of a segment: 4 or 16 a thread. Few rows are cut finer, so that they reach all SMs; many rows coarser, since
// every segment reads its row's history (rows of 201,088 with 1,024 and with 4,096 entries: one 12 and 16 us, two 14 and 18,
// four 16 and 18, twelve 25 and 20, sixty-four 78 and 47, by events around a graph).
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
__device__ __noinline__ float bias_sum(const int* all_ids, const float* all, int biases, int begin, int i, int listed, const int* ids,
                                       const int* places, const float* values) {
    float sum = 0.f;
    if (listed > kLogitsListed) {
        for (int j = 0; j < biases; ++j)
            if (all_ids[j] - begin == i) sum = __fadd_rn(sum, all[j]);
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

template <typename T, int kSegment> __global__ void __launch_bounds__(kLogitsThreads, 5) k_logits(LogitsArgs a) {
    constexpr int kPer = 16 / sizeof(T);
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
            if (c & kBiasBit) x = __fadd_rn(x, bias_sum(a.bias_ids + row * a.bias_ids_stride, a.bias + row * a.bias_stride, a.biases, begin, i, s_listed, listed_ids, listed_at, listed));
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
