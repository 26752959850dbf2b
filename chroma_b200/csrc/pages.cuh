// The pages of a cache: a step of its sequences (continue, fork, empty, reserve, copy before a write) and compaction.
//
// Both are decided on the device from the table and the lengths alone: a page is held iff some slot's rows lie in it,
// so there are no reference counts to keep, and a page that nobody holds is free. Free pages are given out from the
// lowest number to slots from the lowest, so the result does not depend on the order in which CTAs run.
#pragma once

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
};

// One layer's pools and the layout of a page: `rows` rows of `heads` runs of `run` 16-byte words, the strides in
// 16-byte words.
struct PoolArgs {
    uint4 *k, *v;
    int64_t kl, kp, kr, kh, vl, vp, vr, vh;
    int layers, heads, run;
};

__device__ __forceinline__ int pages_of(int rows, int page) { return rows / page + (rows % page != 0); }

struct SlotStep { int parent, old_rows, new_rows; };

__device__ __forceinline__ SlotStep slot_step(const StepArgs& a, int slot) {
    SlotStep s{a.parents[slot], 0, 0};
    if (s.parent < 0 || s.parent >= a.slots) s.parent = -1;
    if (s.parent >= 0) {
        s.old_rows = held_rows(a.lengths, s.parent, a.width, a.page);
        const int64_t want = int64_t(s.old_rows) + max(0, a.counts[slot]), most = int64_t(a.width) * a.page;
        s.new_rows = int(want < most ? want : most);
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

// New table rows from the parents', and each page's keeper: the holder with the most rows in it, then the lowest slot.
__global__ void __launch_bounds__(256) k_pages_gather(StepArgs a) {
    const int slot = blockIdx.y, m = blockIdx.x * 256 + threadIdx.x;
    const SlotStep s = slot_step(a, slot);
    if (m == 0) a.new_lengths[slot] = s.new_rows;
    if (m >= a.width) return;
    int id = -1;
    const int64_t begin = int64_t(m) * a.page;
    if (begin < s.old_rows) {
        id = a.table[s.parent * a.ts + m];
        if (id < 0 || id >= a.pages) id = -1;
        if (id >= 0) {
            const unsigned used = unsigned(min(int64_t(a.page), s.old_rows - begin));
            atomicMax(&a.keeper[id], used * unsigned(a.slots) + unsigned(a.slots - 1 - slot) + 1u);
        }
    }
    a.new_table[int64_t(slot) * a.width + m] = id;
}

// One CTA: the list of free pages, then every slot's share of it.
__global__ void __launch_bounds__(1024) k_pages_assign(StepArgs a) {
    __shared__ int warp_sums[32];
    __shared__ int s_copies;
    if (threadIdx.x == 0) s_copies = 0;
    int nfree = 0, total;
    for (int base = 0; base < a.pages; base += 1024) {
        const int p = base + threadIdx.x;
        const int mine = p < a.pages && a.keeper[p] == 0;
        const int upto = block_scan(mine, warp_sums, &total);
        if (mine) a.free_list[nfree + upto - 1] = p;
        nfree += total;
    }
    __syncthreads();
    int taken = 0;
    for (int base = 0; base < a.slots; base += 1024) {
        const int slot = base + threadIdx.x;
        SlotStep s{-1, 0, 0};
        int copy = 0, fresh = 0, held = 0, source = -1;
        int* row = a.new_table + int64_t(slot) * a.width;
        if (slot < a.slots) {
            s = slot_step(a, slot);
            held = pages_of(s.old_rows, a.page);
            fresh = pages_of(s.new_rows, a.page) - held;
            const int part = s.old_rows % a.page;
            if (part && s.new_rows > s.old_rows) {
                source = row[held - 1];
                copy = source >= 0 && a.keeper[source] != unsigned(part) * unsigned(a.slots) + unsigned(a.slots - 1 - slot) + 1u;
            }
        }
        const int upto = block_scan(copy + fresh, warp_sums, &total);
        int at = taken + upto - copy - fresh;
        if (copy) {
            const int target = at < nfree ? a.free_list[at] : -1;
            ++at;
            row[held - 1] = target;
            int* c = a.copies + 3 * atomicAdd(&s_copies, 1);
            c[0] = source;
            c[1] = target;
            c[2] = s.old_rows % a.page;
        }
        for (int j = 0; j < fresh; ++j, ++at) row[held + j] = at < nfree ? a.free_list[at] : -1;
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

// The first rows of page `source` of every layer's keys and values to page `target`, for each entry of a list in
// device memory.
__global__ void __launch_bounds__(256) k_pages_copy(PoolArgs a, const int* list, const int* count) {
    const int n = *count;
    for (int64_t item = blockIdx.x; item < int64_t(n) * a.layers * 2; item += gridDim.x) {
        const int c = int(item / (2 * a.layers)), layer = int(item % (2 * a.layers)) >> 1;
        const bool value = item & 1;
        const int64_t source = list[3 * c], target = list[3 * c + 1];
        const int words = list[3 * c + 2] * a.heads * a.run;
        uint4* pool = (value ? a.v : a.k) + layer * (value ? a.vl : a.kl);
        const int64_t sp = value ? a.vp : a.kp, sr = value ? a.vr : a.kr, sh = value ? a.vh : a.kh;
        for (int w = threadIdx.x; w < words; w += 256) {
            const int row = w / (a.heads * a.run), rest = w % (a.heads * a.run);
            const int64_t off = row * sr + (rest / a.run) * sh + rest % a.run;
            pool[target * sp + off] = pool[source * sp + off];
        }
    }
}

struct CompactArgs {
    const int* table;
    int64_t ts;
    const int* lengths;
    int *new_table, *info;
    unsigned* held;    // [pages]
    int* to;           // [pages] new number of a held page
    int* copies;       // [pages][3] and the count behind it
    int slots, width, pages, page;
};

__global__ void __launch_bounds__(256) k_compact_mark(CompactArgs a) {
    const int slot = blockIdx.y, m = blockIdx.x * 256 + threadIdx.x;
    if (m >= a.width || int64_t(m) * a.page >= held_rows(a.lengths, slot, a.width, a.page)) return;
    const int id = a.table[slot * a.ts + m];
    if (id >= 0 && id < a.pages) a.held[id] = 1;
}

__global__ void __launch_bounds__(1024) k_compact_plan(CompactArgs a) {
    __shared__ int warp_sums[32];
    int n = 0, total;
    for (int base = 0; base < a.pages; base += 1024) {
        const int p = base + threadIdx.x;
        block_scan(p < a.pages && a.held[p], warp_sums, &total);
        n += total;
    }
    int holes = 0;
    for (int base = 0; base < n; base += 1024) {
        const int p = base + threadIdx.x;
        const int mine = p < n && !a.held[p];
        const int upto = block_scan(mine, warp_sums, &total);
        if (mine) a.copies[3 * (holes + upto - 1) + 1] = p;
        if (p < n && !mine) a.to[p] = p;
        holes += total;
    }
    __syncthreads();
    int moved = 0;
    for (int base = n; base < a.pages; base += 1024) {
        const int p = base + threadIdx.x;
        const int mine = p < a.pages && a.held[p];
        const int upto = block_scan(mine, warp_sums, &total);
        if (mine) {
            int* c = a.copies + 3 * (moved + upto - 1);
            c[0] = p;
            c[2] = a.page;
            a.to[p] = c[1];
        }
        moved += total;
    }
    if (threadIdx.x == 0) {
        a.copies[3 * a.pages] = moved;
        a.info[0] = n;
        a.info[1] = moved;
    }
}

__global__ void __launch_bounds__(256) k_compact_table(CompactArgs a) {
    const int slot = blockIdx.y, m = blockIdx.x * 256 + threadIdx.x;
    if (m >= a.width) return;
    int id = -1;
    if (int64_t(m) * a.page < held_rows(a.lengths, slot, a.width, a.page)) id = a.table[slot * a.ts + m];
    a.new_table[int64_t(slot) * a.width + m] = id >= 0 && id < a.pages ? a.to[id] : -1;
}

}  // namespace cb200
