// What is done to logits before a token is chosen from them: penalties for tokens that occurred, biases, temperature,
// the mask of a grammar, and the greedy choice.
//
// One CTA takes a segment of one row: it counts the row's history into a table of its segment in shared memory, adds the
// biases of its segment in list order, and passes over the logits once, 16 bytes a thread at a time. No table of counts is
// kept between calls. The arithmetic is rounded operation by operation (no fused multiply-add), so that results do not
// depend on how the compiler groups it, and equal logits stay equal. The best of each segment is left for a second, small
// launch. Bound by HBM where there are many rows; a single row by the latency of its few dependent reads.
#pragma once

#include "common.cuh"

namespace cb200 {

// Entries of a segment: 4 or 16 a thread. Few rows are cut finer, so that they reach all SMs; many rows coarser, since
// every segment reads its row's history (a row of 201,088: 24.6 us with 4,096 entries, XXX with 1,024).
constexpr int kLogitsThreads = 256, kLogitsShort = 4 * kLogitsThreads, kLogitsLong = 16 * kLogitsThreads;
constexpr unsigned kHeardBit = 0x80000000u;  // the token occurs in the prompt; the bits below count later occurrences

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
    int vector;  // rows of logits and out are 16-byte aligned
};

template <typename T, int kSegment> __global__ void __launch_bounds__(kLogitsThreads) k_logits(LogitsArgs a) {
    constexpr int kPer = 16 / sizeof(T);
    __shared__ __align__(16) unsigned counts[kSegment];
    __shared__ __align__(16) float added[kSegment];
    __shared__ float listed[32];
    __shared__ unsigned long long keys[kLogitsThreads / 32];
    asm volatile("griddepcontrol.launch_dependents;" :::);
    const int row = blockIdx.y, begin = blockIdx.x * kSegment, n = min(kSegment, a.vocab - begin);
    const float r = a.repetition ? a.repetition[row] : 1.f, f = a.frequency ? a.frequency[row] : 0.f;
    const float pr = a.presence ? a.presence[row] : 0.f, temp = a.temperature ? a.temperature[row] : 0.f;
    const bool heard = a.history, biased = a.bias_ids;
    for (int i = 4 * threadIdx.x; i < kSegment; i += 4 * kLogitsThreads) {
        if (heard) *reinterpret_cast<uint4*>(counts + i) = make_uint4(0, 0, 0, 0);
        if (biased) *reinterpret_cast<float4*>(added + i) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();
    if (heard) {
        const int len = min(max(a.lengths[row], 0), a.width), prompt = a.prompts ? a.prompts[row] : 0;
        const int* history = a.history + row * a.history_stride;
#pragma unroll 4
        for (int i = threadIdx.x; i < len; i += kLogitsThreads) {
            const unsigned t = unsigned(__ldg(history + i) - begin);
            if (t >= unsigned(n)) continue;
            if (i < prompt) atomicOr(&counts[t], kHeardBit);
            else atomicAdd(&counts[t], 1u);
        }
    }
    if (biased && threadIdx.x < 32) {
        for (int base = 0; base < a.biases; base += 32) {
            const int i = base + threadIdx.x;
            int t = i < a.biases ? a.bias_ids[row * a.bias_ids_stride + i] - begin : -1;
            if (t < 0 || t >= n) t = -1;
            listed[threadIdx.x] = t >= 0 ? a.bias[row * a.bias_stride + i] : 0.f;
            const unsigned same = __match_any_sync(0xffffffffu, t);
            __syncwarp();
            if (t >= 0 && (same & ((1u << threadIdx.x) - 1)) == 0) {  // the first of its token adds them all in order
                float sum = added[t];
                for (unsigned rest = same; rest; rest &= rest - 1) sum = __fadd_rn(sum, listed[__ffs(rest) - 1]);
                added[t] = sum;
            }
            __syncwarp();
        }
    }
    __syncthreads();
    const T* in = static_cast<const T*>(a.logits) + row * a.stride + begin;
    T* out = static_cast<T*>(a.out) + row * a.out_stride + begin;
    const unsigned* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    float top = -INFINITY;  // of this thread's entries, and where: the first of equals, the first NaN before all
    int where = -1;
    const auto one = [&](float x, int i, unsigned c, float plus, unsigned allowed) {
        if (c) {
            x = x > 0.f ? __fdiv_rn(x, r) : __fmul_rn(x, r);
            const unsigned times = c & ~kHeardBit;
            if (times) x = __fsub_rn(__fsub_rn(x, __fmul_rn(f, float(times))), pr);
        }
        x = __fadd_rn(x, plus);
        if (temp != 0.f) x = __fdiv_rn(x, temp);
        x = allowed ? Store<T>::round(x) : -INFINITY;
        if (!(x <= top) && top == top) {
            top = x;
            where = i;
        }
        return x;
    };
    if (a.vector) {
        const int first = kPer * threadIdx.x;
        if (first < n) where = first;
#pragma unroll 4
        for (int i = first; i < n; i += kPer * kLogitsThreads) {
            const unsigned allowed = mask ? __ldg(mask + ((begin + i) >> 5)) >> ((begin + i) & 31) : ~0u;
            if (i + kPer <= n) {
                alignas(16) T x[kPer];
                alignas(16) unsigned c[kPer] = {};
                alignas(16) float plus[kPer] = {};
                *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(in + i);
#pragma unroll
                for (int e = 0; e < kPer; e += 4) {
                    if (heard) *reinterpret_cast<uint4*>(c + e) = *reinterpret_cast<const uint4*>(counts + i + e);
                    if (biased) *reinterpret_cast<float4*>(plus + e) = *reinterpret_cast<const float4*>(added + i + e);
                }
#pragma unroll
                for (int e = 0; e < kPer; ++e) Store<T>::store(x + e, one(Store<T>::load(x + e), i + e, c[e], plus[e], allowed >> e & 1));
                *reinterpret_cast<uint4*>(out + i) = *reinterpret_cast<const uint4*>(x);
            } else
                for (int e = 0; i + e < n; ++e)
                    Store<T>::store(out + i + e, one(Store<T>::load(in + i + e), i + e, heard ? counts[i + e] : 0u, biased ? added[i + e] : 0.f, allowed >> e & 1));
        }
    } else {
        if (int(threadIdx.x) < n) where = threadIdx.x;
        for (int i = threadIdx.x; i < n; i += kLogitsThreads) {
            const unsigned allowed = mask ? __ldg(mask + ((begin + i) >> 5)) >> ((begin + i) & 31) & 1 : 1u;
            Store<T>::store(out + i, one(Store<T>::load(in + i), i, heard ? counts[i] : 0u, biased ? added[i] : 0.f, allowed));
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
