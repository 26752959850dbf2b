// A paged key-value cache: what its operators share, the write of new rows, and the attention of any token over the
// pages of its sequence.
//
// Position p of slot s is row p % page of page table[s][p / page] of the pools. A token at position p sees position j
// iff j <= p, j's page exists, and p - j < window or j < first (no window: every j <= p). All sums and the softmax's
// maximum are kept in fp32.
#pragma once

#include "common.cuh"

namespace cb200 {

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery, "Division by invariant integers using
// multiplication", 1994): l = ceil(log2 d), m = floor(2^32 (2^l - d) / d) + 1, q = (mulhi(m, n) + n) >> l.
struct FastDiv {
    uint32_t d = 1, m = 1, l = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t divisor) : d(divisor) {
        while ((uint64_t(1) << l) < d) ++l;
        m = uint32_t((((uint64_t(1) << l) - d) << 32) / d + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(m, n) + n) >> l; }
};

struct PagedArgs {
    const void *k, *v;              // pools
    int64_t kp, kr, kh, vp, vr, vh; // elements between pages, rows, heads
    const int* table;
    int64_t ts;                     // elements between table rows
    const int* lengths;
    const int* starts;              // nullptr: one token per slot
    int slots, width, pages, page, kv, dim;
    FastDiv by_page;
    const void* q;
    void* out;
    float* lse;
    const void* sinks;
    int64_t qt, qh, ot, oh;         // elements between tokens, heads
    int tokens, heads, group, sinks_fp32, window, first;
    float scale_log2;               // scale * log2(e)
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Rows a slot holds, within what its table can name.
__device__ __forceinline__ int held_rows(const int* lengths, int slot, int width, int page) {
    const int64_t most = int64_t(width) * page;
    const int n = lengths[slot];
    return n < 0 ? 0 : int64_t(n) > most ? int(most) : n;
}

// Slot of a token: the last slot whose first row is not after it, or -1 (rows before the first slot or past the last).
__device__ __forceinline__ int slot_of(const int* starts, int slots, int token) {
    int lo = 0, hi = slots;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid + 1] <= token) lo = mid + 1;
        else hi = mid;
    }
    return lo < slots && starts[lo] <= token ? lo : -1;
}

// The learned sink of a head in the log2 domain; -inf where there is none.
template <typename T> __device__ __forceinline__ float sink_log2(const void* sinks, int fp32, int head) {
    if (!sinks) return -INFINITY;
    return (fp32 ? static_cast<const float*>(sinks)[head] : Store<T>::load(static_cast<const T*>(sinks) + head)) * kLog2e;
}

__device__ __forceinline__ bool sees(int p, int j, int window, int first) {
    return j <= p && (window <= 0 || p - j < window || j < first);
}

struct AppendArgs {
    const void *nk, *nv;
    int64_t nkt, nkh, nvt, nvh;     // elements between tokens, heads of the new rows
    void *k, *v;
    int64_t kp, kr, kh, vp, vr, vh;
    const int* table;
    int64_t ts;
    const int* lengths;
    const int* starts;
    int slots, width, pages, page, kv, dim, tokens;
    FastDiv by_page;
};

// 16-byte words of new rows to their pages, kAppendTokens tokens a CTA: the places of its tokens are looked up once, a thread
// each, then all threads copy. `vector`: source rows are 16-byte aligned (the pools always are). Bound by HBM, and by the
// three dependent reads (starts, lengths, table) where there are few tokens.
constexpr int kAppendTokens = 8;
template <typename T> __global__ void __launch_bounds__(256) k_paged_append(AppendArgs a, int vector) {
    __shared__ int64_t places[kAppendTokens][2];
    const int token0 = blockIdx.x * kAppendTokens;
    if (threadIdx.x < kAppendTokens) {
        const int token = token0 + threadIdx.x;
        int64_t kplace = -1, vplace = -1;
        const int slot = token >= a.tokens ? -1 : a.starts ? slot_of(a.starts, a.slots, token) : token;
        if (slot >= 0) {
            const int len = held_rows(a.lengths, slot, a.width, a.page);
            const int pos = a.starts ? len - a.starts[slot + 1] + token : len - 1;
            if (pos >= 0) {
                const int entry = int(a.by_page.div(uint32_t(pos))), id = a.table[slot * a.ts + entry];
                if (id >= 0 && id < a.pages) {
                    kplace = id * a.kp + (pos - entry * a.page) * a.kr;
                    vplace = id * a.vp + (pos - entry * a.page) * a.vr;
                }
            }
        }
        places[threadIdx.x][0] = kplace;
        places[threadIdx.x][1] = vplace;
    }
    __syncthreads();
    constexpr int kPer = 16 / sizeof(T);
    const int run = a.dim / kPer, words = a.kv * run;  // of a token's keys, or values
#pragma unroll 4
    for (int e = threadIdx.x; e < kAppendTokens * 2 * words; e += 256) {
        const int t = e / (2 * words), rest = e % (2 * words), value = rest >= words, w = rest - value * words;
        const int h = w / run, d = (w - h * run) * kPer, token = token0 + t;
        const int64_t place = places[t][value];
        if (place < 0) continue;
        const T* from = static_cast<const T*>(value ? a.nv : a.nk) + token * (value ? a.nvt : a.nkt) + h * (value ? a.nvh : a.nkh) + d;
        T* to = static_cast<T*>(value ? a.v : a.k) + place + h * (value ? a.vh : a.kh) + d;
        if (vector) *reinterpret_cast<uint4*>(to) = __ldg(reinterpret_cast<const uint4*>(from));
        else
#pragma unroll
            for (int i = 0; i < kPer; ++i) to[i] = from[i];
    }
}

}  // namespace cb200
