// The pages of a cache: a step of its sequences (continue, fork, empty, reserve, copy before a write) and compaction.
//
// Both are decided on the device from the table and the lengths alone: a page is held iff some slot's rows lie in it,
// so there are no reference counts to keep, and a page that nobody holds is free. Free pages are given out from the
// lowest number to slots from the lowest, so the result does not depend on the order in which CTAs run.
//
// The decision is a chain of dependent passes over slots, pages and table entries, and bound by their latency: one CTA in
// shared memory where all fits there (4,096 pages, 128 slots: 10 us), a few small launches otherwise. The copies are bound by
// HBM: compaction of 64 sequences of 500-2,500 in four layers (1 GB moved) takes 172-180 us in all, 5.7 TB/s.
#pragma once

#include <limits.h>

#include "paged.cuh"

namespace cb200 {

struct StepArgs {
    const int* table;
    int64_t ts;
    const int *lengths, *parents, *counts;
    int *new_table, *new_lengths, *info;
    unsigned* keeper;   // [pages] 0: free; else 1 + rows used * slots + (slots - 1 - slot) of the page's keeper
    int* free_list;     // [pages]
    int* copies;        // [slots][3]: source page, target page, rows; copies[3 * slots]: how many
    int slots, width, pages, page;
    int cut;            // new lengths end where the table does
};

// One layer's pools and the layout of a page: `rows` rows of `heads` runs of `run` 16-byte words, the strides in
// 16-byte words.
struct PoolArgs {
    uint4 *k, *v;
    int64_t kl, kp, kr, kh, vl, vp, vr, vh;
    int layers, heads, run;
};

__device__ __forceinline__ int pages_of(int rows, int page) { return rows / page + (rows % page != 0); }

// old_rows, new_rows: rows within what the table can name.
struct SlotStep { int parent, old_rows, new_rows, new_length; };

__device__ __forceinline__ SlotStep slot_step(const StepArgs& a, int slot) {
    SlotStep s{a.parents[slot], 0, 0, 0};
    if (s.parent < 0 || s.parent >= a.slots) s.parent = -1;
    if (s.parent >= 0) {
        s.old_rows = held_rows(a.lengths, s.parent, a.width, a.page);
        const int64_t more = max(0, a.counts[slot]), want = s.old_rows + more, most = int64_t(a.width) * a.page;
        s.new_rows = int(want < most ? want : most);
        s.new_length = a.cut ? s.new_rows : int(min(length_of(a.lengths, s.parent) + more, int64_t(INT_MAX)));
    }
    return s;
}

// Inclusive prefix sum over a block of 1,024 threads; *total receives the block's sum.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    if (warp == 0) {
        int w = warp_sums[lane];
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += u;
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    *total = warp_sums[31];
    return v + (warp ? warp_sums[warp - 1] : 0);
}

// Entry m of a slot's new table row, from its parent's, and the page's keeper: the holder with the most rows in it, then the
// lowest slot.
__device__ __forceinline__ void gather_entry(const StepArgs& a, const SlotStep& s, unsigned* keeper, int slot, int m) {
    int id = -1;
    const int64_t begin = int64_t(m) * a.page;
    if (begin < s.old_rows) {
        id = a.table[s.parent * a.ts + m];
        if (id < 0 || id >= a.pages) id = -1;
        if (id >= 0) {
            const unsigned used = unsigned(min(int64_t(a.page), s.old_rows - begin));
            atomicMax(&keeper[id], used * unsigned(a.slots) + unsigned(a.slots - 1 - slot) + 1u);
        }
    }
    a.new_table[int64_t(slot) * a.width + m] = id;
}

[[maybe_unused]] static __global__ void __launch_bounds__(256) k_pages_gather(StepArgs a) {
    const int m = blockIdx.x * 256 + threadIdx.x;
    const SlotStep s = slot_step(a, blockIdx.y);
    if (m == 0) a.new_lengths[blockIdx.y] = s.new_length;
    if (m < a.width) gather_entry(a, s, a.keeper, blockIdx.y, m);
}

// One CTA of 1,024: the numbers of the pages for which pick(p) holds, in ascending order, through put(rank, p). Returns how
// many there are.
template <typename Pick, typename Put>
__device__ __forceinline__ int list_pages(int pages, int* warp_sums, Pick&& pick, Put&& put) {
    const int per = (pages + 1023) / 1024, p0 = threadIdx.x * per, p1 = min(pages, p0 + per);
    int mine = 0, total;
    for (int p = p0; p < p1; ++p) mine += pick(p);
    int rank = block_scan(mine, warp_sums, &total) - mine;
    for (int p = p0; p < p1; ++p)
        if (pick(p)) put(rank++, p);
    return total;
}

// One CTA: the list of free pages, then every slot's share of it.
template <typename List, typename Slot>
__device__ __forceinline__ void assign_pages(const StepArgs& a, const unsigned* keeper, List* free_list, Slot&& slot_at) {
    __shared__ int warp_sums[32];
    __shared__ int s_copies;
    if (threadIdx.x == 0) s_copies = 0;
    int total;
    const int nfree = list_pages(a.pages, warp_sums, [&](int p) { return keeper[p] == 0; }, [&](int rank, int p) { free_list[rank] = List(p); });
    __syncthreads();
    int taken = 0;
    for (int base = 0; base < a.slots; base += 1024) {
        const int slot = base + threadIdx.x;
        SlotStep s{-1, 0, 0, 0};
        int copy = 0, fresh = 0, held = 0, source = -1;
        int* row = a.new_table + int64_t(slot) * a.width;
        if (slot < a.slots) {
            s = slot_at(slot);
            held = pages_of(s.old_rows, a.page);
            fresh = pages_of(s.new_rows, a.page) - held;
            const int part = s.old_rows % a.page;
            if (part && s.new_rows > s.old_rows) {
                source = row[held - 1];
                copy = source >= 0 && keeper[source] != unsigned(part) * unsigned(a.slots) + unsigned(a.slots - 1 - slot) + 1u;
            }
        }
        const int upto = block_scan(copy + fresh, warp_sums, &total);
        int at = taken + upto - copy - fresh;
        if (copy) {
            const int target = at < nfree ? int(free_list[at]) : -1;
            ++at;
            row[held - 1] = target;
            int* c = a.copies + 3 * atomicAdd(&s_copies, 1);
            c[0] = source;
            c[1] = target;
            c[2] = s.old_rows % a.page;
        }
        for (int j = 0; j < fresh; ++j, ++at) row[held + j] = at < nfree ? int(free_list[at]) : -1;
        taken += total;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        const int lacking = max(0, taken - nfree);
        // Nothing is copied by a step that lacks pages: its inputs and every page they name stay as they were.
        const int n = lacking ? 0 : s_copies;
        a.copies[3 * a.slots] = n;
        a.info[0] = max(0, nfree - taken);
        a.info[1] = lacking;
        a.info[2] = n;
    }
}

[[maybe_unused]] static __global__ void __launch_bounds__(1024) k_pages_assign(StepArgs a) {
    asm volatile("griddepcontrol.launch_dependents;" :::);
    assign_pages(a, a.keeper, a.free_list, [&](int slot) { return slot_step(a, slot); });
}

// The whole decision in one CTA, in shared memory: the keepers [pages], what becomes of the slots [slots], the free list.
[[maybe_unused]] static __global__ void __launch_bounds__(1024) k_pages_step(StepArgs a) {
    extern __shared__ unsigned page_marks[];
    SlotStep* steps = reinterpret_cast<SlotStep*>(page_marks + a.pages);
    asm volatile("griddepcontrol.launch_dependents;" :::);
    for (int slot = threadIdx.x; slot < a.slots; slot += 1024) {
        const SlotStep s = slot_step(a, slot);
        steps[slot] = s;
        a.new_lengths[slot] = s.new_length;
    }
    for (int p = threadIdx.x; p < a.pages; p += 1024) page_marks[p] = 0;
    __syncthreads();
#pragma unroll 4
    for (int e = threadIdx.x; e < a.slots * a.width; e += 1024) gather_entry(a, steps[e / a.width], page_marks, e / a.width, e % a.width);
    __syncthreads();
    assign_pages(a, page_marks, reinterpret_cast<uint16_t*>(steps + a.slots), [&](int slot) { return steps[slot]; });
}

// The first rows of page `source` of every layer's keys and values to page `target`, for each entry (source, target, rows)
// of a list in device memory: 16 KB a CTA at a time, four words a thread under way.
[[maybe_unused]] static __global__ void __launch_bounds__(256) k_pages_copy(PoolArgs a, const int* list, const int* count) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int row_words = a.heads * a.run, part = blockIdx.y;  // 1,024 words of a page
    const bool plain = a.heads == 1 && a.kr == a.run && a.vr == a.run;  // a page is one run
    const int64_t total = int64_t(*count) * a.layers * 2;
    for (int64_t item = blockIdx.x; item < total; item += gridDim.x) {
        const unsigned c = unsigned(item) / unsigned(2 * a.layers), layer = unsigned(item) % unsigned(2 * a.layers) >> 1;
        const bool value = item & 1;
        const int words = list[3 * c + 2] * row_words, w0 = part * 1024 + threadIdx.x;
        if (part * 1024 >= words) continue;
        const int64_t sp = value ? a.vp : a.kp, sr = value ? a.vr : a.kr, sh = value ? a.vh : a.kh;
        uint4* pool = (value ? a.v : a.k) + layer * (value ? a.vl : a.kl);
        const uint4* from = pool + list[3 * c] * sp;
        uint4* to = pool + list[3 * c + 1] * sp;
        int64_t off[4];
        uint4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int w = w0 + i * 256;
            off[i] = plain ? w : w / row_words * sr + w % row_words / a.run * sh + w % a.run;
            if (w < words) x[i] = from[off[i]];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (w0 + i * 256 < words) to[off[i]] = x[i];
    }
}

struct CompactArgs {
    const int* table;
    int64_t ts;
    const int* lengths;
    int *new_table, *info;
    unsigned* held;    // [pages] marks; then 1 + the new number of a held page
    int* copies;       // [pages][3] and the count behind it
    int* holes;        // [pages]
    int slots, width, pages, page;
};

__device__ __forceinline__ int held_entry(const CompactArgs& a, int slot, int m) {  // the page there, or -1
    if (int64_t(m) * a.page >= held_rows(a.lengths, slot, a.width, a.page)) return -1;
    const int id = a.table[slot * a.ts + m];
    return id >= 0 && id < a.pages ? id : -1;
}

// One CTA: held[p] becomes 1 + the new number of each held page; the list of moves. `holes` [pages]: scratch.
template <typename List> __device__ __forceinline__ void plan_moves(const CompactArgs& a, unsigned* held, List* holes) {
    __shared__ int warp_sums[32];
    int n;
    {
        const int per = (a.pages + 1023) / 1024, p0 = threadIdx.x * per, p1 = min(a.pages, p0 + per);
        int mine = 0;
        for (int p = p0; p < p1; ++p) mine += held[p] != 0;
        block_scan(mine, warp_sums, &n);
    }
    list_pages(n, warp_sums, [&](int p) { return held[p] == 0; }, [&](int rank, int p) { holes[rank] = List(p); });
    __syncthreads();
    const int moved = list_pages(a.pages - n, warp_sums, [&](int p) { return held[n + p] != 0; }, [&](int rank, int p) {
        const int to = int(holes[rank]);
        a.copies[3 * rank] = n + p;
        a.copies[3 * rank + 1] = to;
        a.copies[3 * rank + 2] = a.page;
        held[n + p] = unsigned(to) + 1;
    });
    for (int p = threadIdx.x; p < n; p += 1024)
        if (held[p]) held[p] = p + 1;
    if (threadIdx.x == 0) {
        a.copies[3 * a.pages] = moved;
        a.info[0] = n;
        a.info[1] = moved;
    }
}

__device__ __forceinline__ void renumber_entry(const CompactArgs& a, const unsigned* held, int slot, int m) {
    const int id = held_entry(a, slot, m);
    a.new_table[int64_t(slot) * a.width + m] = id >= 0 ? int(held[id]) - 1 : -1;
}

[[maybe_unused]] static __global__ void __launch_bounds__(256) k_compact_mark(CompactArgs a) {
    const int m = blockIdx.x * 256 + threadIdx.x, id = m < a.width ? held_entry(a, blockIdx.y, m) : -1;
    if (id >= 0) a.held[id] = 1;
}
[[maybe_unused]] static __global__ void __launch_bounds__(1024) k_compact_plan(CompactArgs a) { plan_moves(a, a.held, a.holes); }
[[maybe_unused]] static __global__ void __launch_bounds__(256) k_compact_table(CompactArgs a) {
    const int m = blockIdx.x * 256 + threadIdx.x;
    asm volatile("griddepcontrol.launch_dependents;" :::);
    if (m < a.width) renumber_entry(a, a.held, blockIdx.y, m);
}

// The whole decision in one CTA, in shared memory: the marks [pages], the holes [pages]. A thread's first entries stay in
// registers from the marking to the renumbering.
[[maybe_unused]] static __global__ void __launch_bounds__(1024) k_compact(CompactArgs a) {
    extern __shared__ unsigned page_marks[];
    constexpr int kKept = 4;
    asm volatile("griddepcontrol.launch_dependents;" :::);
    int ids[kKept];
    const int entries = a.slots * a.width;
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
        const int e = threadIdx.x + i * 1024;
        ids[i] = e < entries ? held_entry(a, e / a.width, e % a.width) : -1;
    }
    for (int p = threadIdx.x; p < a.pages; p += 1024) page_marks[p] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kKept; ++i)
        if (ids[i] >= 0) page_marks[ids[i]] = 1;
    for (int e = threadIdx.x + kKept * 1024; e < entries; e += 1024) {
        const int id = held_entry(a, e / a.width, e % a.width);
        if (id >= 0) page_marks[id] = 1;
    }
    __syncthreads();
    plan_moves(a, page_marks, reinterpret_cast<uint16_t*>(page_marks + a.pages));
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kKept; ++i) {
        const int e = threadIdx.x + i * 1024;
        if (e < entries) a.new_table[e] = ids[i] >= 0 ? int(page_marks[ids[i]]) - 1 : -1;
    }
    for (int e = threadIdx.x + kKept * 1024; e < entries; e += 1024) renumber_entry(a, page_marks, e / a.width, e % a.width);
}

}  // namespace cb200
