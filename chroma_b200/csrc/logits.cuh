// What is done to logits before a token is chosen from them: penalties for tokens that occurred, biases, temperature,
// the mask of a grammar, and the greedy choice.
//
// One CTA takes kLogitsSegment entries of one row: it counts the row's history into a table of its segment in shared
// memory, adds the biases of its segment in list order, and passes over the logits once. No table of counts is kept
// between calls. The arithmetic is rounded operation by operation (no fused multiply-add), so that results do not
// depend on how the compiler groups it.
#pragma once

#include "common.cuh"

namespace cb200 {

constexpr int kLogitsSegment = 4096;
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
};

template <typename T> __global__ void __launch_bounds__(256) k_logits(LogitsArgs a) {
    __shared__ unsigned counts[kLogitsSegment];
    __shared__ float added[kLogitsSegment];
    __shared__ float listed[32];
    __shared__ unsigned long long keys[8];
    const int row = blockIdx.y, begin = blockIdx.x * kLogitsSegment, n = min(kLogitsSegment, a.vocab - begin);
    for (int i = threadIdx.x; i < kLogitsSegment; i += 256) {
        counts[i] = 0;
        added[i] = 0.f;
    }
    __syncthreads();
    if (a.history) {
        const int len = min(max(a.lengths[row], 0), a.width), prompt = a.prompts ? a.prompts[row] : 0;
        for (int i = threadIdx.x; i < len; i += 256) {
            const int t = a.history[row * a.history_stride + i] - begin;
            if (t < 0 || t >= n) continue;
            if (i < prompt) atomicOr(&counts[t], kHeardBit);
            else atomicAdd(&counts[t], 1u);
        }
    }
    if (a.bias_ids && threadIdx.x < 32) {
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
    const float r = a.repetition ? a.repetition[row] : 1.f, f = a.frequency ? a.frequency[row] : 0.f;
    const float pr = a.presence ? a.presence[row] : 0.f, temp = a.temperature ? a.temperature[row] : 0.f;
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int v = begin + i;
        float x = Store<T>::load(static_cast<const T*>(a.logits) + row * a.stride + v);
        const unsigned c = counts[i];
        if (c) {
            x = x > 0.f ? __fdiv_rn(x, r) : __fmul_rn(x, r);
            const unsigned times = c & ~kHeardBit;
            if (times) x = __fsub_rn(__fsub_rn(x, __fmul_rn(f, float(times))), pr);
        }
        x = __fadd_rn(x, added[i]);
        if (temp != 0.f) x = __fdiv_rn(x, temp);
        if (a.mask && !((a.mask[row * a.mask_stride + (v >> 5)] >> (v & 31)) & 1u)) x = -INFINITY;
        x = Store<T>::round(x);
        Store<T>::store(static_cast<T*>(a.out) + row * a.out_stride + v, x);
        const unsigned long long key = argmax_key(x + 0.0f, v);  // + 0: a negative zero equals a positive one
        best = key > best ? key : best;
    }
    if (!a.best) return;
    for (int o = 16; o; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
        best = other > best ? other : best;
    }
    if ((threadIdx.x & 31) == 0) keys[threadIdx.x >> 5] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) best = keys[w] > best ? keys[w] : best;
        a.best[int64_t(row) * a.segments + blockIdx.x] = best;
    }
}

// The best of a row's segments; one warp per row.
[[maybe_unused]] static __global__ void __launch_bounds__(32) k_logits_pick(const unsigned long long* best, int segments,
                                                                           int64_t* argmax) {
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
