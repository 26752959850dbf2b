// A paged key-value cache: what its operators share, and the write of new rows.
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

// Length of a slot: one past its last token's position, which may lie past what its table can name.
__device__ __forceinline__ int length_of(const int* lengths, int slot) { return max(lengths[slot], 0); }

// Rows a slot holds, within what its table can name.
__device__ __forceinline__ int held_rows(const int* lengths, int slot, int width, int page) {
    const int64_t most = int64_t(width) * page;
    const int n = length_of(lengths, slot);
    return int64_t(n) > most ? int(most) : n;
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
    FastDiv by_page, by_run;        // by_run.d: 16-byte words of a head's row
};

// New rows to their pages, a warp per token, 16 bytes a lane. The warp's first words are read while its token's place is looked
// up; up to 256 slots are all compared with the token at once (one read deep), more are searched. `vector`: source rows are
// 16-byte aligned (the pools always are). Bound by HBM, and by the three dependent reads (starts and lengths, table, then the
// stores) where there are few tokens: 18,544 rows of 2 KB in each pool 16 us, 4.7 TB/s; 128 rows 4.1 us, of which the host's
// call takes 3.2.
constexpr int kAppendWarps = 8;
template <typename T> __global__ void __launch_bounds__(32 * kAppendWarps) k_paged_append(AppendArgs a, int vector) {
    constexpr int kPer = 16 / sizeof(T), kAtOnce = 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, token = blockIdx.x * kAppendWarps + warp;
    if (token >= a.tokens) return;
    const int words = a.kv * int(a.by_run.d), total = 2 * words;  // words of the token's keys, then of its values
    const T *nk = static_cast<const T*>(a.nk) + token * a.nkt, *nv = static_cast<const T*>(a.nv) + token * a.nvt;
    const auto split = [&](int e, int& value, int& h, int& d) {
        value = e >= words;
        const int w = e - value * words;
        h = int(a.by_run.div(w));
        d = (w - h * int(a.by_run.d)) * kPer;
    };
    uint4 x[kAtOnce];
    const auto load = [&](int e0) {
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            int value, h, d;
            const int e = e0 + 32 * i;
            split(e, value, h, d);
            if (e < total) x[i] = __ldg(reinterpret_cast<const uint4*>((value ? nv + h * a.nvh : nk + h * a.nkh) + d));
        }
    };
    if (vector) load(lane);
    int slot = token, pos = -1;
    if (a.starts && a.slots <= 256) {
        int found = -1;
#pragma unroll 4
        for (int s = lane; s < a.slots; s += 32) {
            const int first = a.starts[s], end = a.starts[s + 1], length = length_of(a.lengths, s);
            if (first <= token && token < end) {
                found = s;
                pos = length - end + token;
            }
        }
        const unsigned who = __ballot_sync(0xffffffffu, found >= 0);
        if (!who) return;
        slot = __shfl_sync(0xffffffffu, found, __ffs(who) - 1);
        pos = __shfl_sync(0xffffffffu, pos, __ffs(who) - 1);
    } else {
        if (a.starts) slot = slot_of(a.starts, a.slots, token);
        if (slot < 0) return;
        pos = length_of(a.lengths, slot) - (a.starts ? a.starts[slot + 1] - token : 1);
    }
    if (pos < 0) return;
    const int entry = int(a.by_page.div(uint32_t(pos)));
    if (entry >= a.width) return;
    const int id = a.table[slot * a.ts + entry];
    if (id < 0 || id >= a.pages) return;
    T* k = static_cast<T*>(a.k) + id * a.kp + (pos - entry * a.page) * a.kr;
    T* v = static_cast<T*>(a.v) + id * a.vp + (pos - entry * a.page) * a.vr;
    for (int e0 = lane; e0 < total; e0 += 32 * kAtOnce) {
        if (vector && e0 != lane) load(e0);
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            int value, h, d;
            const int e = e0 + 32 * i;
            split(e, value, h, d);
            if (e >= total) continue;
            T* to = (value ? v + h * a.vh : k + h * a.kh) + d;
            if (vector) *reinterpret_cast<uint4*>(to) = x[i];
            else {
                const T* from = (value ? nv + h * a.nvh : nk + h * a.nkh) + d;
#pragma unroll
                for (int c = 0; c < kPer; ++c) to[c] = from[c];
            }
        }
    }
}

}  // namespace cb200
