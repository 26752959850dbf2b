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

// One warp per (token, head): 32 keys at a time, one per lane, then the values of the visible ones, one after another.
// Right for every type, shape and mask.
template <typename T> __global__ void __launch_bounds__(128) k_paged_attention_rows(PagedArgs a) {
    extern __shared__ float rows_q[];  // [4][dim]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t item = int64_t(blockIdx.x) * 4 + warp;
    if (item >= int64_t(a.tokens) * a.heads) return;
    const int token = int(item / a.heads), head = int(item % a.heads), kvh = head / a.group;
    const int slot = a.starts ? slot_of(a.starts, a.slots, token) : token;
    if (slot < 0) return;
    const int len = held_rows(a.lengths, slot, a.width, a.page);
    const int pos = a.starts ? len - a.starts[slot + 1] + token : len - 1;
    float* q = rows_q + warp * a.dim;
    const T* qrow = static_cast<const T*>(a.q) + token * a.qt + head * a.qh;
    for (int d = lane; d < a.dim; d += 32) q[d] = Store<T>::load(qrow + d);
    __syncwarp();
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    const int low = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const int first = min(a.first, low);  // [0, first) then [low, pos]
    const int total = max(0, pos + 1 - low + first);
    for (int base = 0; base < total; base += 32) {
        const int i = base + lane;
        const int j = i < first ? i : low + i - first;
        const int entry = i < total ? int(a.by_page.div(uint32_t(j))) : 0;
        int id = i < total ? a.table[slot * a.ts + entry] : -1;
        if (id >= a.pages) id = -1;
        float s = -INFINITY;
        const int row = j - entry * a.page;
        if (id >= 0) {
            const T* k = static_cast<const T*>(a.k) + id * a.kp + row * a.kr + kvh * a.kh;
            float dot = 0.f;
            for (int d = 0; d < a.dim; ++d) dot = fmaf(q[d], Store<T>::load(k + d), dot);
            s = dot * a.scale_log2;
        }
        const float mx = fmaxf(m, warp_max(s));
        if (mx == -INFINITY && !__any_sync(0xffffffffu, id >= 0 && isnan(s))) continue;
        const float corr = m == -INFINITY ? 0.f : exp2f(m - mx);
        const float p = id < 0 ? 0.f : exp2f(s - mx);
        l = l * corr + warp_sum(p);
        m = mx;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] *= corr;
        for (int e = 0; e < min(32, total - base); ++e) {
            const int ide = __shfl_sync(0xffffffffu, id, e), rowe = __shfl_sync(0xffffffffu, row, e);
            const float pe = __shfl_sync(0xffffffffu, p, e);
            if (ide < 0) continue;
            const T* v = static_cast<const T*>(a.v) + ide * a.vp + rowe * a.vr + kvh * a.vh;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (c * 32 + lane < a.dim) o[c] = fmaf(pe, Store<T>::load(v + c * 32 + lane), o[c]);
        }
    }
    const float sink = sink_log2<T>(a.sinks, a.sinks_fp32, head);
    const float top = fmaxf(m, sink);
    const float c = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2f(m - top);
    const float sum = l * c + (sink == -INFINITY ? 0.f : exp2f(sink - top));
    T* orow = static_cast<T*>(a.out) + token * a.ot + head * a.oh;
    for (int d = lane; d < a.dim; d += 32) Store<T>::store(orow + d, sum == 0.f ? 0.f : o[d >> 5] * c / sum);
    if (a.lse && lane == 0) a.lse[item] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
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

// One CTA per token: its key and value heads to their page, element by element.
template <typename T> __global__ void __launch_bounds__(128) k_paged_append(AppendArgs a) {
    const int token = blockIdx.x;
    const int slot = a.starts ? slot_of(a.starts, a.slots, token) : token;
    if (slot < 0) return;
    const int len = held_rows(a.lengths, slot, a.width, a.page);
    const int pos = a.starts ? len - a.starts[slot + 1] + token : len - 1;
    if (pos < 0) return;
    const int entry = int(a.by_page.div(uint32_t(pos)));
    const int id = a.table[slot * a.ts + entry];
    if (id < 0 || id >= a.pages) return;
    const int row = pos - entry * a.page;
    for (int e = threadIdx.x; e < a.kv * a.dim; e += blockDim.x) {
        const int h = e / a.dim, d = e % a.dim;
        static_cast<T*>(a.k)[id * a.kp + row * a.kr + h * a.kh + d] = static_cast<const T*>(a.nk)[token * a.nkt + h * a.nkh + d];
        static_cast<T*>(a.v)[id * a.vp + row * a.vr + h * a.vh + d] = static_cast<const T*>(a.nv)[token * a.nvt + h * a.nvh + d];
    }
}

}  // namespace cb200
