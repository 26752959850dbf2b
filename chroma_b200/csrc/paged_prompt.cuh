// Attention of prompts over a paged cache on the 5th-generation tensor cores (bf16): chunks of any lengths, each after
// what its sequence's pages hold already, causal, with a sliding window that keeps the first positions in sight.
//
// A row is one query head of one token; the rows of a key-value head are packed, token after token with its `group`
// query heads side by side, so that a tile of 128 rows shares every key even where a chunk has few tokens. A work item
// is 256 consecutive rows (two tiles) of one key-value head of one sequence, against key tiles of 128 positions. The
// grid is persistent, one CTA per SM; items with the most keys before them come first, the key-value heads of the same rows
// side by side. 12 warps:
//   warps 0-3, 4-7  the online softmax of tile 0, 1, one row per thread (TMEM lane = row): the row of S (128 columns)
//                   from TMEM at once, P = 2^(s - m) back over its first 64 columns as bf16 pairs; at the item's end
//                   O / l to global memory
//   warp 8          one thread issues, per key tile t and tile k in turn: O_k += P_k(t) V(t), S_k(t+1) = Q_k K(t+1)^T
//   warp 9          K and V tiles into a ring, by TMA boxes of as many rows as divide the page (a box never leaves its
//                   page), or, where the pool or the page size is none that TMA takes, row by row with cp.async
//   warps 10, 11    Q of tile 0, 1 of the next item, as soon as the last S of this one is done
// P stays in tensor memory as the A operand of the product with V. Heads of up to 64 values leave room for P beside S, so
// that S_k(t+1) is computed while the exponentials of S_k(t) are taken. With wider heads P lies over S: the tensor core
// runs the products of one issuing thread in order, so S_k(t+1) lands only after O_k has taken P_k(t), and the commit
// that signals S_k(t+1) covers that product too. The maximum moves only when a tile exceeds it by more than 2^8, so O is
// rescaled rarely.
//
// What bounds it: the exponentials and what goes with them on 128 rows of one thread each, in turn with the products
// (clock stamps per tile of 64-value heads: 1,400 cycles of exponentials, 650 around them, 1,000 waiting; the
// special-function unit is busy half of the time, the tensor core a quarter). Four prompts of 2,048 tokens, 64/8 heads of
// 64: 283 us, 486 TFLOP/s (269 one call after another); 8,192 tokens after 8,001 in a window of 4,096, 32/8 heads of 128:
// 586 us, 939 TFLOP/s, and 628 to 636 once the GPU is at its power limit; two prompts of 4,096 with 32/8 heads of 128: 297 us. No unit
// is full: issue slots 36 and 29% (heads of 64, 128), the special-function unit 52 and 44%, the tensor core 25 and 44%.
// Tried when those two took 300 and 586 us, and slower: a quarter to a half of the exponentials as a polynomial on the FMA
// pipe (305 to 354 us, though issue slots are not short; why was not found), the issuing warp taking whatever is ready first
// (301 and 653 us), a second issuing warp (317 and 640 us), the two tiles' exponentials in turn (313 and 604 us).
//
// A position that no row may see costs nothing (whole tiles are passed over) or a mask of 128 bits per row, applied only
// to the tiles that need it. Values behind the end of a sequence are cleared in shared memory, since what lies there may
// not be finite. Positions that some rows of a tile see and others do not meet the others with weight 0, which is no
// protection against infinities: a CTA that finds one in a result takes its items a second time, with such values cleaned.
//
// Where there are few items (a short chunk after a long cache), the keys of each are split over several CTAs, which leave
// fp32 partial results for k_prompt_join (16 tokens after 16,000, 64/8 heads of 64: 69 us, without splits 203).
//
// All waits are bounded (tma.cuh).
#pragma once

#include <type_traits>

#include "paged_decode.cuh"

namespace cb200 {

constexpr int kPrThreads = 384, kPrTile = 128;
constexpr int kPrSorted = 1024, kPrSortedSlots = 64;  // pairs of tiles and slots that are put in order
// Registers of a softmax thread and of the others, out of the 3 x 168 that three warpgroups are launched with.
constexpr int kPrSoftmaxRegs = 216, kPrOtherRegs = 72;

// The products are issued by one elected thread of a converged warp: everything they need is the same in all lanes, so it
// can stay in uniform registers (issued from a branch that one lane takes, a step cost up to twice its time).
//
// Four steps of 16 along K of D[tmem] (+)= A[smem] B[smem]^T over one 64-value block (K-major, 128-byte swizzle), as one
// statement: the steps' descriptors are constants apart, and nothing comes between the instructions.
__device__ __forceinline__ void umma_ss_block(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q, e;\n\t.reg .b64 a1, a2, a3, b1, b2, b3;\n\telect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 q, 0, 0;\n\t"
        "add.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"
        "add.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, q;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(accumulate))
        : "memory");
}

// Eight steps of 16 along K of D[tmem] (+)= P[tmem] V[smem]: P 128 x 128 (8 columns a step), V MN-major (2 KB a step).
__device__ __forceinline__ void umma_ts_128(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q, e;\n\t.reg .b64 b1, b2, b3, b4, b5, b6, b7;\n\t.reg .b32 a1, a2, a3, a4, a5, a6, a7;\n\telect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 q, 0, 0;\n\t"
        "add.s64 b1, %2, 128;\n\tadd.s64 b2, %2, 256;\n\tadd.s64 b3, %2, 384;\n\tadd.s64 b4, %2, 512;\n\t"
        "add.s64 b5, %2, 640;\n\tadd.s64 b6, %2, 768;\n\tadd.s64 b7, %2, 896;\n\t"
        "add.s32 a1, %1, 8;\n\tadd.s32 a2, %1, 16;\n\tadd.s32 a3, %1, 24;\n\tadd.s32 a4, %1, 32;\n\t"
        "add.s32 a5, %1, 40;\n\tadd.s32 a6, %1, 48;\n\tadd.s32 a7, %1, 56;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a4], b4, %3, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a5], b5, %3, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a6], b6, %3, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a7], b7, %3, q;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(accumulate))
        : "memory");
}

// Arrives on `bar` once the products that the elected thread issued before are done.
__device__ __forceinline__ void umma_commit_elected(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar))
        : "memory");
}

struct PagedPromptArgs {
    PagedArgs a;
    FastDiv by_group, by_kv;
    int box;                 // rows of a TMA box; 0: row by row
    int q_vector, out_vector;  // rows are 16-byte aligned
    int q_box;               // Q tiles come as one TMA box: `group` heads of 128 / group tokens
    int over_q;              // results are written over Q: no second time, the first is taken like it
    int tiles;               // pairs of tiles of rows at most: what the workspace has room for
    int splits;              // of the keys of an item, where there are few items
    FastDiv by_splits;
    float* parts;            // [items][splits][256 rows][64 H]: what the splits of a row come to, unless there is one
    float2* part_ml;         // [items][splits][256 rows]: maximum (log2 domain) and sum
    unsigned* error;
};

// 64 H values per row (H = 1, 2): Q tiles, then a ring of K and V tiles, in blocks of [128 rows][64 values] with the
// 128-byte swizzle; then each stage's missing positions.
template <int H> struct PromptShape {
    static constexpr int kBlock = kPrTile * 128, kTile = H * kBlock, kStage = 2 * kTile, kStages = H == 2 ? 2 : 4;
    static constexpr int kSmem = 1024 + 2 * kTile + kStages * kStage + kStages * 16;
};

// A work item: 256 rows of one key-value head of one slot, and the key tiles that they see.
struct PromptItem {
    int slot, kvh, row0, rows, token0, pos0;  // first row; rows of the slot; first token; its position
    int tiles, skip, pre, main0;              // key tiles of the split, after `skip`: of [0, pre), then from main0 on
    int active;                               // tiles of rows: 1 or 2
    int64_t part;                             // number of this split's first row
    unsigned number;                          // of all splits of all items
    __device__ __forceinline__ int key0(int t) const { return (skip + t < pre ? skip + t : main0 + skip + t - pre) * kPrTile; }
};

__device__ __forceinline__ uint32_t* prompt_order() {
    __shared__ uint32_t order[kPrSorted];
    return order;
}

// The items of a CTA in turn: blockIdx.x, + gridDim.x (backwards every other round, which evens out their sizes), ...
struct PromptCursor {
    int slot, before, round;  // tiles of the slots after `slot`
    bool sorted;              // or prompt_order() has slot << 16 | tile of each place
    bool second = false;      // the second time, or the only one
    __device__ __forceinline__ explicit PromptCursor(const PagedArgs& a, bool in_order = false)
        : slot(a.slots - 1), before(0), round(0), sorted(in_order) {}
    // The end of the first time, for every warp of the CTA.
    static __device__ __forceinline__ void end_first() {
        __syncwarp();
        asm volatile("bar.sync 1, %0;" ::"n"(kPrThreads) : "memory");
    }
    // After the last item: back to the first if `bad` says so by then.
    __device__ __forceinline__ bool again(const PagedPromptArgs& p, const volatile int& bad) {
        if (second) return false;
        second = true;
        end_first();
        slot = p.a.slots - 1;
        before = round = 0;
        return bad;
    }
    static __device__ __forceinline__ int rows_of(const PagedArgs& a, int s) {
        const int t0 = min(max(a.starts[s], 0), a.tokens), t1 = min(max(a.starts[s + 1], 0), a.tokens);
        return max(0, t1 - t0) * a.group;
    }
    // Adds up the pairs of tiles of all slots. Rows that a falling `starts` gives to several slots are counted for each, so the
    // sum may pass what the host made room for: callers cut it there.
    static __device__ __forceinline__ void count_tiles(const PagedArgs& a, unsigned long long* sum) {
        unsigned long long mine = 0;
        for (int s = threadIdx.x; s < a.slots; s += blockDim.x) mine += (rows_of(a, s) + 255) / 256;
        if (mine) atomicAdd(sum, mine);
    }
    __device__ __forceinline__ bool next(const PagedPromptArgs& p, int total, PromptItem& w) {
        const unsigned i = unsigned(round) * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        ++round;
        if (i >= unsigned(total) * unsigned(p.a.kv) * unsigned(p.splits)) return false;
        take(p, i, w);
        return true;
    }
    // Number i of all splits of all items.
    __device__ __forceinline__ void take(const PagedPromptArgs& p, unsigned i, PromptItem& w) {
        find(p, p.splits == 1 ? i : p.by_splits.div(i), w);
        if (p.splits > 1) {
            const int z = int(i - p.by_splits.div(i) * unsigned(p.splits)), all = w.tiles;
            w.skip = int(int64_t(all) * z / p.splits);
            w.tiles = int(int64_t(all) * (z + 1) / p.splits) - w.skip;
            w.part = int64_t(i) * 256;
        }
        w.number = i;
    }
    // Item i of all (a later one than the last).
    __device__ __forceinline__ void find(const PagedPromptArgs& p, unsigned i, PromptItem& w) {
        const PagedArgs& a = p.a;
        const int tile = int(p.by_kv.div(i));
        w.kvh = int(i) - tile * a.kv;
        int rows;
        if (sorted) {
            const uint32_t place = prompt_order()[tile];
            slot = int(place >> 16);
            rows = rows_of(a, slot);
            w.row0 = int(place & 0xffff) * 256;
        } else {
            rows = rows_of(a, slot);
            int n = (rows + 255) / 256;
            while (tile >= before + n) {
                before += n;
                --slot;
                rows = rows_of(a, slot);
                n = (rows + 255) / 256;
            }
            w.row0 = (n - 1 - (tile - before)) * 256;
        }
        w.slot = slot;
        w.rows = rows;
        w.token0 = min(max(a.starts[slot], 0), a.tokens);
        w.pos0 = length_of(a.lengths, slot) - rows / a.group;
        w.active = w.row0 + kPrTile < rows ? 2 : 1;
        const int first = w.pos0 + int(p.by_group.div(w.row0)), last = w.pos0 + int(p.by_group.div(min(w.row0 + 256, rows) - 1));
        const int low = a.window > 0 ? max(0, first - a.window + 1) : 0, top = min(last, a.width * a.page - 1);
        w.pre = (min(a.first, min(low, top + 1)) + kPrTile - 1) / kPrTile;
        w.main0 = max(low / kPrTile, w.pre);
        w.tiles = last < 0 ? 0 : w.pre + max(0, top / kPrTile - w.main0 + 1);
        w.skip = 0;
        w.part = 0;
    }
};

// ---- Values that are not finite. A weight of 0 does not keep them from a row that does not see them. So where a row's result is
// not finite although its sum of weights is (a score that is not finite makes the sum so, and belongs to a key that the row sees,
// since others are replaced), the CTA takes its items a second time. Then the values of tiles of keys that not every row of a
// tile sees are cleaned in shared memory, and each row is given what it sees of them afterwards. The second time costs as much
// as the first, and a pass over the values of those tiles: 600 tokens after 6,000, 16/8 heads of 64, 0.1 ms and 0.7 with one bad
// value among them; computing such rows again one by one, while the pipeline waited, took 112.
//
// Everything for the second time is inlined and takes its arguments anew from the item's number: calls from the loop over the
// items, though never made, cost the first time 2 to 4% (four prompts of 2,048: 293 us for 283).

// Whether every row of tile k of an item sees every position of the tile of keys at j0.
__device__ __forceinline__ bool whole_tile(const PagedPromptArgs& p, const PromptItem& w, int k, int j0) {
    const int first = w.pos0 + int(p.by_group.div(w.row0 + k * kPrTile));
    const int last = w.pos0 + int(p.by_group.div(min(w.row0 + (k + 1) * kPrTile, w.rows) - 1));
    return j0 + kPrTile - 1 <= first && (p.a.window <= 0 || last - j0 < p.a.window || j0 + kPrTile <= p.a.first);
}

__device__ __forceinline__ bool has_bad(const uint4& x) {
    const auto bad = [](uint32_t v) { return (v & 0x7f80) == 0x7f80 || (v & 0x7f800000) == 0x7f800000; };
    return bad(x.x) || bad(x.y) || bad(x.z) || bad(x.w);
}
__device__ __forceinline__ uint32_t cleaned(uint32_t x) {
    return ((x & 0x7f80) == 0x7f80 ? 0u : x & 0xffffu) | ((x & 0x7f800000) == 0x7f800000 ? 0u : x & 0xffff0000u);
}

// Row r of a tile of values in shared memory without what is not finite; true if there was something.
template <int H> __device__ __forceinline__ bool clean_row(uint8_t* tile, int r) {
    bool found = false;
    for (int c = 0; c < 8 * H; ++c) {
        uint4* at = reinterpret_cast<uint4*>(tile + (c >> 3) * PromptShape<H>::kBlock + r * 128 + (((c ^ r) & 7) << 4));
        uint4 x = *at;
        if (!has_bad(x)) continue;
        found = true;
        *at = make_uint4(cleaned(x.x), cleaned(x.y), cleaned(x.z), cleaned(x.w));
    }
    return found;
}

// A softmax thread's row of item `number`.
template <int H> struct SecondLook {
    PromptItem w;
    int pos = -1;
    __nv_bfloat16* out = nullptr;  // the row's result, or its part of a split's
    float* part = nullptr;
    __device__ __forceinline__ SecondLook(const PagedPromptArgs& p, unsigned number, bool sorted) {
        PromptCursor(p.a, sorted).take(p, number, w);
        const int row = w.row0 + threadIdx.x, n = int(p.by_group.div(row));
        if (row >= w.rows) return;
        pos = w.pos0 + n;
        out = static_cast<__nv_bfloat16*>(p.a.out) + (w.token0 + n) * p.a.ot + (w.kvh * p.a.group + row - n * p.a.group) * p.a.oh;
        part = p.splits > 1 ? p.parts + (w.part + threadIdx.x) * (64 * H) : nullptr;
    }
};

// Adds to a thread's row what it sees of the values that were cleaned.
template <int H> __device__ __forceinline__ void add_cleaned(const PagedPromptArgs& p, unsigned number, bool sorted) {
    const PagedArgs& a = p.a;
    const SecondLook<H> look(p, number, sorted);
    const PromptItem& w = look.w;
    bool done = look.pos < 0;  // no row, or nothing but NaN
#pragma unroll 1
    for (int t = 0; t < w.tiles; ++t) {
        const int t0 = w.key0(t);
        if (whole_tile(p, w, 0, t0) && (w.active == 1 || whole_tile(p, w, 1, t0))) continue;
#pragma unroll 1
        for (int j = t0; j < t0 + kPrTile; ++j) {
            if (__all_sync(0xffffffffu, done)) return;
            int nans = 0;
            const int entry = int(a.by_page.div(uint32_t(j))), id = entry < a.width ? __ldg(a.table + w.slot * a.ts + entry) : -1;
            if (id < 0 || id >= a.pages) continue;
            const auto* v = static_cast<const __nv_bfloat16*>(a.v) + id * a.vp + (j - entry * a.page) * a.vr + w.kvh * a.vh;
#pragma unroll 1
            for (int d = 0; d < a.dim; d += 8) {
                if (!has_bad(__ldg(reinterpret_cast<const uint4*>(v + d))) || done || !sees(look.pos, j, a.window, a.first)) continue;
#pragma unroll 1
                for (int e = d; e < d + 8; ++e) {
                    const float x = __bfloat162float(v[e]);
                    if (x * 0.f == 0.f) continue;
                    nans += isnan(x);
                    const float was = look.part ? look.part[e] : __bfloat162float(look.out[e]);
                    if (was == x) continue;  // an infinity more
                    if (look.part) look.part[e] = was + x;
                    else look.out[e] = __float2bfloat16_rn(was + x);
                }
            }
            done = done || nans == a.dim;
        }
    }
}

__device__ __forceinline__ uint32_t bits_from_to(int lo, int hi) {  // bits lo..hi of a word, cut to it
    lo = max(lo, 0);
    hi = min(hi, 31);
    return hi < lo ? 0u : (0xffffffffu >> (31 - hi)) & (0xffffffffu << lo);
}

template <int H>
__global__ void __launch_bounds__(kPrThreads, 1)
k_paged_prompt(const __grid_constant__ PagedPromptArgs p, const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
               const __grid_constant__ CUtensorMap vmap) {
    using Shape = PromptShape<H>;
    // TMEM columns: S of the two tiles; P of each over its S (H = 2) or in 64 columns of its own (H = 1); O.
    constexpr bool kOwnP = H == 1;
    constexpr int kStages = Shape::kStages, D = 64 * H, kO = 512 - 2 * D;
    extern __shared__ uint8_t pr_raw[];
    asm volatile("griddepcontrol.launch_dependents;" :::);
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(pr_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* Qs = sm;                           // [2][H][128][64]
    uint8_t* KV = Qs + 2 * Shape::kTile;        // stage s: K at s * kStage, V kTile behind it
    uint32_t* gone = reinterpret_cast<uint32_t*>(KV + kStages * Shape::kStage);  // [kStages][4]
    __shared__ uint64_t q_full[2], q_empty[2], kv_full[kStages], kv_empty[kStages], s_full[2], s_free[2], p_full[2], o_done[2];
    __shared__ uint32_t tmem_base;
    __shared__ int tile_counts[kPrSortedSlots];
    __shared__ unsigned long long s_total;
    __shared__ volatile int abort_flag, bad_flag, cleaned_flag;  // bad_flag: a result is not finite; cleaned_flag: a value was cleaned
    const PagedArgs& a = p.a;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int k = 0; k < 2; ++k) {
            mbar_init(&q_full[k], 1);
            mbar_init(&q_empty[k], 1);
            mbar_init(&s_full[k], 1);
            mbar_init(&s_free[k], 4);
            mbar_init(&p_full[k], 4);
            mbar_init(&o_done[k], 1);
        }
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&kv_full[s], 1);
            mbar_init(&kv_empty[s], 1);
        }
        abort_flag = bad_flag = cleaned_flag = 0;
        s_total = 0;
        fence_barrier_init();
    }
    if (warp == 8) {
        tmem_alloc(&tmem_base, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    PromptCursor::count_tiles(a, &s_total);
    __syncthreads();
    const int total = int(min(s_total, (unsigned long long)p.tiles));
    const uint32_t tmem = tmem_base;
    // With few sequences their tiles are put in order, the later (with more keys before them) first, whatever the sequence:
    // four prompts of 2,048 tokens are then within 1% of an even load, against 10% in the order of the sequences.
    const bool sorted = p.splits == 1 && s_total <= kPrSorted && a.slots <= kPrSortedSlots;
    if (sorted) {
        for (int s = threadIdx.x; s < a.slots; s += kPrThreads) tile_counts[s] = (PromptCursor::rows_of(a, s) + 255) / 256;
        __syncthreads();
        for (int e = threadIdx.x; e < int(s_total); e += kPrThreads) {
            int slot = 0, tile = e, place = 0;
            while (tile >= tile_counts[slot]) tile -= tile_counts[slot++];
            for (int s = 0; s < a.slots; ++s) place += max(0, tile_counts[s] - 1 - tile) + (s < slot && tile_counts[s] > tile);
            prompt_order()[place] = uint32_t(slot) << 16 | uint32_t(tile);
        }
        __syncthreads();
    }

    if (warp >= 8) {
    PromptCursor cursor(a, sorted);
    cursor.second = p.over_q;
    PromptItem w;
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPrOtherRegs));
    if (warp == 9) {
        // ---- K and V
        int g = 0;  // tiles so far
        while (!abort_flag) {
            if (!cursor.next(p, total, w)) {
                if (cursor.again(p, bad_flag)) continue;
                break;
            }
            for (int t = 0; t < w.tiles; ++t, ++g) {
                const int s = g % kStages;
                if (!mbar_wait(&kv_empty[s], unsigned((g / kStages) & 1) ^ 1, p.error)) abort_flag = 1;
                if (abort_flag) break;
                const int j0 = w.key0(t);
                uint8_t* kd = KV + s * Shape::kStage;
                if (lane < 4) gone[s * 4 + lane] = 0;
                __syncwarp();
                if (p.box) {
                    const int boxes = kPrTile / p.box;
                    int row = 0, id = a.pages;  // beyond the map: zeros
                    if (lane < boxes) {
                        const int j = j0 + lane * p.box, entry = int(a.by_page.div(uint32_t(j)));
                        row = j - entry * a.page;
                        if (entry < a.width) id = __ldg(a.table + w.slot * a.ts + entry);
                        if (id < 0 || id >= a.pages) {
                            id = a.pages;
                            for (int e = lane * p.box; e < (lane + 1) * p.box; e += 8)
                                atomicOr(&gone[s * 4 + (e >> 5)], 0xffu << (e & 31));
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive_expect_tx(&kv_full[s], Shape::kStage);
                    __syncwarp();
                    if (lane < boxes)
#pragma unroll
                        for (int h = 0; h < H; ++h) {
                            uint8_t* to = kd + h * Shape::kBlock + lane * p.box * 128;
                            asm volatile(
                                "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_addr(to)),
                                "l"(reinterpret_cast<uint64_t>(&kmap)), "r"(h * 64), "r"(w.kvh), "r"(row), "r"(id), "r"(smem_addr(&kv_full[s]))
                                : "memory");
                            asm volatile(
                                "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_addr(to + Shape::kTile)),
                                "l"(reinterpret_cast<uint64_t>(&vmap)), "r"(h * 64), "r"(w.kvh), "r"(row), "r"(id), "r"(smem_addr(&kv_full[s]))
                                : "memory");
                        }
                } else {
                    const int end = held_rows(a.lengths, w.slot, a.width, a.page);
                    for (int base = 0; base < kPrTile; base += 32) {  // a row per lane, its address handed round
                        const int j = j0 + base + lane, entry = int(a.by_page.div(uint32_t(j)));
                        int id = j < end ? __ldg(a.table + w.slot * a.ts + entry) : -1;
                        if (id >= a.pages) id = -1;
                        const int row = j - entry * a.page;
                        const uint32_t none = __ballot_sync(0xffffffffu, id < 0);
                        if (lane == 0) gone[s * 4 + (base >> 5)] = none;
                        const int64_t ko = id < 0 ? 0 : id * a.kp + row * a.kr + w.kvh * a.kh;
                        const int64_t vo = id < 0 ? 0 : id * a.vp + row * a.vr + w.kvh * a.vh;
                        constexpr int kChunks = 8 * H, kRows = 32 / kChunks;  // 16-byte chunks of a row, rows at a time
                        for (int r0 = 0; r0 < 32; r0 += kRows) {
                            const int r = r0 + lane / kChunks, c = lane % kChunks;
                            const int64_t kr = __shfl_sync(0xffffffffu, ko, r), vr = __shfl_sync(0xffffffffu, vo, r);
                            const bool ok = !(none >> r & 1) && c * 8 < a.dim;
                            uint8_t* to = kd + (c >> 3) * Shape::kBlock + (base + r) * 128 + (((c & 7) ^ (r & 7)) << 4);
                            const auto* ks = static_cast<const __nv_bfloat16*>(a.k) + kr + (ok ? c * 8 : 0);
                            const auto* vs = static_cast<const __nv_bfloat16*>(a.v) + vr + (ok ? c * 8 : 0);
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(to)), "l"(ks), "r"(ok ? 16 : 0) : "memory");
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(to + Shape::kTile)), "l"(vs), "r"(ok ? 16 : 0) : "memory");
                        }
                    }
                    cp_async_commit();
                    cp_async_wait<0>();
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&kv_full[s]);
                }
            }
        }
        if (!cursor.second) cursor.end_first();
        if (abort_flag)  // after a wait that gave up: the copies under way end (or are given up) before the memory is left
            for (int i = max(0, g - kStages); i < g; ++i)
                if (!mbar_wait(&kv_full[i % kStages], unsigned((i / kStages) & 1), p.error)) break;
    } else if (warp >= 10) {
        // ---- Q of tile `warp - 10`
        const int k = warp - 10;
        int loads = 0;
        while (!abort_flag) {
            if (!cursor.next(p, total, w)) {
                if (cursor.again(p, bad_flag)) continue;
                break;
            }
            if (!w.tiles || k >= w.active) continue;
            if (!mbar_wait(&q_empty[k], unsigned(loads & 1) ^ 1, p.error)) abort_flag = 1;
            if (abort_flag) break;
            ++loads;
            constexpr int kChunks = 8 * H;
            uint8_t* to0 = Qs + k * Shape::kTile;
            const int first = w.row0 + k * kPrTile;
            if (p.q_box) {
                if (lane == 0) {
                    mbar_arrive_expect_tx(&q_full[k], Shape::kTile);
                    for (int h = 0; h < H; ++h)
                        tma_load_3d(to0 + h * Shape::kBlock, &qmap, h * 64, w.kvh * a.group, w.token0 + int(p.by_group.div(first)), &q_full[k]);
                }
                continue;
            }
            for (int e = lane; e < kPrTile * kChunks; e += 32) {
                const int r = e / kChunks, c = e % kChunks, row = first + r;
                const int token = int(p.by_group.div(row)), head = w.kvh * a.group + row - token * a.group;
                const bool ok = row < w.rows && c * 8 < a.dim;
                uint8_t* to = to0 + (c >> 3) * Shape::kBlock + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                const auto* from = static_cast<const __nv_bfloat16*>(a.q) + (ok ? (w.token0 + token) * a.qt + head * a.qh + c * 8 : 0);
                if (p.q_vector)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(to)), "l"(from), "r"(ok ? 16 : 0) : "memory");
                else
                    for (int i = 0; i < 8; ++i)
                        reinterpret_cast<uint16_t*>(to)[i] = ok ? reinterpret_cast<const uint16_t*>(from)[i] : uint16_t(0);
            }
            cp_async_commit();
            cp_async_wait<0>();
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[k]);
        }
        if (!cursor.second) cursor.end_first();
        if (abort_flag && loads) mbar_wait(&q_full[k], unsigned(loads - 1) & 1, p.error);
    } else if (warp == 8) {
        // ---- products, ping-pong over the two tiles of rows; the warp stays converged
        constexpr uint32_t idesc_s = umma_idesc_bf16(kPrTile, kPrTile);
        constexpr uint32_t idesc_o = umma_idesc_bf16(kPrTile, D) | (1u << 16);  // B (V) MN-major
        int g = 0, q_used[2] = {0, 0}, s_used[2] = {0, 0}, p_used[2] = {0, 0};
        const auto wait = [&](uint64_t* bar, int n) {
            const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, unsigned(n & 1), p.error));
            if (!ok) abort_flag = 1;
            tc_fence_after();
            return ok;
        };
        // S_k of tile t of the item: over columns that have been read (own columns for P) or whose P has been used.
        const auto next_s = [&](int k, int tile, int t) {
            if (kOwnP && s_used[k] && !wait(&s_free[k], s_used[k] - 1)) return false;
            ++s_used[k];
            const uint64_t dq = umma_desc_sw128(Qs + k * Shape::kTile);
            const uint64_t dk = umma_desc_sw128(KV + (tile % kStages) * Shape::kStage);
#pragma unroll
            for (int h = 0; h < H; ++h)
                umma_ss_block(tmem + uint32_t(k * kPrTile), dq + h * (Shape::kBlock >> 4), dk + h * (Shape::kBlock >> 4), idesc_s, h > 0);
            umma_commit_elected(&s_full[k]);
            if (t + 1 == w.tiles) umma_commit_elected(&q_empty[k]);
            return true;
        };
        const auto next_o = [&](int k, int tile, int t) {
            const uint64_t dv = umma_desc_sw128_mn(KV + (tile % kStages) * Shape::kStage + Shape::kTile, Shape::kBlock);
            if (!wait(&p_full[k], p_used[k])) return false;
            umma_ts_128(tmem + uint32_t(kO + k * D), tmem + uint32_t(kOwnP ? 2 * kPrTile + k * 64 : k * kPrTile), dv, idesc_o, t > 0);
            ++p_used[k];
            if (kOwnP || t + 1 == w.tiles) umma_commit_elected(&o_done[k]);
            if (k == w.active - 1) umma_commit_elected(&kv_empty[tile % kStages]);
            return true;
        };
        while (!abort_flag) {
            if (!cursor.next(p, total, w)) {
                if (cursor.again(p, bad_flag)) continue;
                break;
            }
            if (!w.tiles) continue;
            const bool two = w.active == 2;
            bool ok = wait(&kv_full[g % kStages], g / kStages);
            for (int k = 0; k < w.active && ok; ++k) ok = wait(&q_full[k], q_used[k]++) && next_s(k, g, 0);
            for (int t = 0; t < w.tiles && ok; ++t, ++g) {
                const bool more = t + 1 < w.tiles;
                if (kOwnP) {  // the order in which two warpgroups half a period apart get there
                    if (more) ok = wait(&kv_full[(g + 1) % kStages], (g + 1) / kStages);
                    if (ok && more) ok = next_s(0, g + 1, t + 1);
                    if (ok && two && t) ok = next_o(1, g - 1, t - 1);
                    if (ok && two && more) ok = next_s(1, g + 1, t + 1);
                    if (ok) ok = next_o(0, g, t);
                    if (ok && two && !more) ok = next_o(1, g, t);
                } else {
                    for (int k = 0; k < w.active && ok; ++k) {
                        ok = next_o(k, g, t);
                        if (ok && more && k == 0) ok = wait(&kv_full[(g + 1) % kStages], (g + 1) / kStages);
                        if (ok && more) ok = next_s(k, g + 1, t + 1);
                    }
                }
                if (abort_flag) ok = false;
            }
        }
        if (!cursor.second) cursor.end_first();
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPrSoftmaxRegs));
        // ---- softmax of tile k; this warp's TMEM lanes are its rows [32 q, 32 q + 32)
        const int k = warp >> 2, q = warp & 3, r = q * 32 + lane;
        const uint32_t lanes = uint32_t(q * 32) << 16;
        const uint32_t tS = tmem + uint32_t(k * kPrTile) + lanes, tO = tmem + uint32_t(kO + k * D) + lanes;
        const uint32_t tP = kOwnP ? tmem + uint32_t(2 * kPrTile + k * 64) + lanes : tS;
        int g = 0, uses = 0, ends = 0;
        PromptCursor cursor(a, sorted);
        cursor.second = p.over_q;
        PromptItem w;
        while (!abort_flag) {
            if (!cursor.next(p, total, w)) {
                if (cursor.again(p, bad_flag)) continue;
                break;
            }
            if (k >= w.active) {
                g += w.tiles;
                continue;
            }
            const int row = w.row0 + k * kPrTile + r, number = int(p.by_group.div(row));
            const int token = w.token0 + number, head = w.kvh * a.group + row - number * a.group;
            const bool row_ok = row < w.rows;
            const int pos = row_ok ? w.pos0 + number : -1;
            // Positions that every row of the tile sees: [max(low_all, 0), first_all].
            const int pos_first = w.pos0 + int(p.by_group.div(w.row0 + k * kPrTile));
            const int pos_last = w.pos0 + int(p.by_group.div(min(w.row0 + (k + 1) * kPrTile, w.rows) - 1));
            const int end = w.pos0 + w.rows / a.group;  // rows that the slot holds
            const int low = a.window > 0 ? pos - a.window + 1 : 0;
            const float sink = row_ok ? sink_log2<__nv_bfloat16>(a.sinks, a.sinks_fp32, head) : -INFINITY;
            float m_run = -INFINITY, l_run = 0.f;
            for (int t = 0; t < w.tiles; ++t, ++g) {
                const int s = g % kStages, j0 = w.key0(t);
                if (!mbar_wait(&kv_full[s], unsigned((g / kStages) & 1), p.error)) abort_flag = 1;
                const uint4 none = *reinterpret_cast<const uint4*>(gone + s * 4);
                const bool whole = j0 + kPrTile - 1 <= pos_first && (a.window <= 0 || pos_last - j0 < a.window || j0 + kPrTile <= a.first);
                const bool all = whole && !(none.x | none.y | none.z | none.w);
                if (cursor.second && !whole) {
                    if (clean_row<H>(KV + s * Shape::kStage + Shape::kTile, r)) cleaned_flag = 1;
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                if (!mbar_wait(&s_full[k], unsigned(uses++ & 1), p.error)) abort_flag = 1;
                if (abort_flag) break;
                tc_fence_after();
                uint32_t sv[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_load32_async(tS + 32 * c, sv + 32 * c);
                tmem_wait_ld();
                if (kOwnP) {  // S may be overwritten
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_free[k]);
                }
                if (!all) {
                    const uint32_t nw[4] = {none.x, none.y, none.z, none.w};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int base = j0 + 32 * c;
                        const uint32_t vis = (bits_from_to(low - base, pos - base) | bits_from_to(0, min(a.first - 1, pos) - base)) & ~nw[c];
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!((vis >> e) & 1)) sv[32 * c + e] = __float_as_uint(-INFINITY);
                    }
                    if (j0 + r >= end) {  // behind the end of the sequence: no values
#pragma unroll
                        for (int c = 0; c < 8 * H; ++c)
                            *reinterpret_cast<uint4*>(KV + s * Shape::kStage + Shape::kTile + (c >> 3) * Shape::kBlock + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                }
                float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 128; e += 8) {
                    mq[0] = fmax3(mq[0], __uint_as_float(sv[e]), __uint_as_float(sv[e + 1]));
                    mq[1] = fmax3(mq[1], __uint_as_float(sv[e + 2]), __uint_as_float(sv[e + 3]));
                    mq[2] = fmax3(mq[2], __uint_as_float(sv[e + 4]), __uint_as_float(sv[e + 5]));
                    mq[3] = fmax3(mq[3], __uint_as_float(sv[e + 6]), __uint_as_float(sv[e + 7]));
                }
                const float m_tile = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3])) * a.scale_log2;
                const float m_new = m_tile > m_run + 8.f ? m_tile : m_run;
                const float corr = m_run == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
                const float neg = m_new == -INFINITY ? 0.f : -m_new;
                m_run = m_new;
                // P's own columns, and O, are this warpgroup's once the product before is done; without own columns, S said so.
                // Waited for here and not before P is stored, it also keeps the two warpgroups half a period apart (then 300 us
                // for the four prompts of 2,048 tokens, against 334).
                if (kOwnP) {
                    if (uses > 1 && !mbar_wait(&o_done[k], unsigned(uses & 1), p.error)) abort_flag = 1;
                    tc_fence_after();
                }
                const uint64_t scale2 = f32x2(a.scale_log2, a.scale_log2), neg2 = f32x2(neg, neg);
                uint64_t sum2[2] = {f32x2(0.f, 0.f), f32x2(0.f, 0.f)};
                uint32_t pw[64];
#pragma unroll
                for (int u = 0; u < 64; ++u) {
                    const uint64_t x = ffma2(f32x2(__uint_as_float(sv[2 * u]), __uint_as_float(sv[2 * u + 1])), scale2, neg2);
                    float xa, xb;
                    f32x2_split(x, xa, xb);
                    xa = fast_exp2(xa);
                    xb = fast_exp2(xb);
                    sum2[u & 1] = fadd2(sum2[u & 1], f32x2(xa, xb));
                    // The weights go into the product with 8 bits, as bf16 operands have; their sum keeps all.
                    pw[u] = pack_bf16(xa, xb);
                    if (u == 31) tmem_store32_async(tP, pw);
                }
                tmem_store32_async(tP + 32, pw + 32);
                float sa, sb;
                f32x2_split(fadd2(sum2[0], sum2[1]), sa, sb);
                if (t > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        float ov[32];
                        tmem_load32(tO + c * 32, ov);
#pragma unroll
                        for (int e = 0; e < 32; ++e) ov[e] *= corr;
                        tmem_store32(tO + c * 32, ov);
                    }
                }
                tmem_wait_st();
                l_run = l_run * corr + (sa + sb);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[k]);
            }
            if (abort_flag) break;
            // ---- the item's end
            float check = 0.f;  // NaN as soon as something is not finite
            if (p.splits > 1) {
                const int64_t at = w.part + k * kPrTile + r;
                if (w.tiles) {
                    if (!mbar_wait(&o_done[k], unsigned((kOwnP ? uses - 1 : ends++) & 1), p.error)) abort_flag = 1;
                    if (abort_flag) break;
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        float ov[32];
                        tmem_load32(tO + c * 32, ov);
#pragma unroll
                        for (int e = 0; e < 32; ++e) check = fmaf(ov[e], 0.f, check);
#pragma unroll
                        for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(p.parts + at * D + c * 32 + e) = make_float4(ov[e], ov[e + 1], ov[e + 2], ov[e + 3]);
                    }
                    if (row_ok && check != 0.f && l_run * 0.f == 0.f) bad_flag = 1;
                    if (cursor.second && cleaned_flag) add_cleaned<H>(p, w.number, sorted);
                }
                p.part_ml[at] = make_float2(m_run, l_run);
                tc_fence_before();
                continue;
            }
            const float top = fmaxf(m_run, sink);
            const float c0 = m_run == -INFINITY ? (l_run == 0.f ? 0.f : 1.f) : fast_exp2(m_run - top);
            const float sum = l_run * c0 + (sink == -INFINITY ? 0.f : fast_exp2(sink - top));
            const float inv = sum == 0.f ? 0.f : c0 / sum;
            __nv_bfloat16* orow = static_cast<__nv_bfloat16*>(a.out) + token * a.ot + head * a.oh;
            if (w.tiles) {
                if (!mbar_wait(&o_done[k], unsigned((kOwnP ? uses - 1 : ends++) & 1), p.error)) abort_flag = 1;
                if (abort_flag) break;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    float ov[32];
                    tmem_load32(tO + c * 32, ov);
#pragma unroll
                    for (int e = 0; e < 32; ++e) check = fmaf(ov[e], 0.f, check);
                    if (row_ok)
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            const int d = c * 32 + e;
                            if (d >= a.dim) continue;
                            uint32_t w4[4];
#pragma unroll
                            for (int u = 0; u < 4; ++u) w4[u] = pack_bf16(ov[e + 2 * u] * inv, ov[e + 2 * u + 1] * inv);
                            if (p.out_vector) *reinterpret_cast<uint4*>(orow + d) = make_uint4(w4[0], w4[1], w4[2], w4[3]);
                            else
#pragma unroll
                                for (int u = 0; u < 8; ++u) reinterpret_cast<uint16_t*>(orow + d)[u] = uint16_t(w4[u >> 1] >> (16 * (u & 1)));
                        }
                }
                if (row_ok && check != 0.f && l_run * 0.f == 0.f) bad_flag = 1;
                if (cursor.second && cleaned_flag) add_cleaned<H>(p, w.number, sorted);
            } else if (row_ok) {
                for (int d = 0; d < a.dim; ++d) orow[d] = __float2bfloat16_rn(0.f);
            }
            if (a.lse && row_ok) a.lse[int64_t(token) * a.heads + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
            tc_fence_before();  // O has been read before its next products are asked for
        }
        if (!cursor.second) cursor.end_first();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the splits of every row, in their order: a warp per row, 32 rows of an item a CTA.
template <int H> __global__ void __launch_bounds__(256) k_prompt_join(const __grid_constant__ PagedPromptArgs p) {
    constexpr int D = 64 * H;
    __shared__ unsigned long long s_total;
    const PagedArgs& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) s_total = 0;
    __syncthreads();
    PromptCursor::count_tiles(a, &s_total);
    __syncthreads();
    const unsigned i = blockIdx.x >> 3;
    if (i >= unsigned(min(s_total, (unsigned long long)p.tiles)) * unsigned(a.kv)) return;
    PromptCursor cursor(a);
    PromptItem w;
    cursor.find(p, i, w);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int r = (blockIdx.x & 7) * 32 + warp; r < ((blockIdx.x & 7) + 1) * 32; r += 8) {
        const int row = w.row0 + r, number = int(p.by_group.div(row));
        if (row >= w.rows) break;
        const int token = w.token0 + number, head = w.kvh * a.group + row - number * a.group;
        const auto part = [&](int z) { return (int64_t(i) * p.splits + z) * 256 + r; };
        float top = -INFINITY, sum = 0.f, x[D / 32] = {};
        for (int z = lane; z < p.splits; z += 32) top = fmaxf(top, p.part_ml[part(z)].x);
        top = warp_max(top);
        for (int z = 0; z < p.splits; ++z) {
            const float2 ml = p.part_ml[part(z)];
            const float weight = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : fast_exp2(ml.x - top);
            if (weight == 0.f) continue;
            sum += ml.y * weight;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) x[c] += p.parts[part(z) * D + c * 32 + lane] * weight;
        }
        const HeadEnd end = head_end(top, sum, sink_log2<__nv_bfloat16>(a.sinks, a.sinks_fp32, head));
        __nv_bfloat16* orow = static_cast<__nv_bfloat16*>(a.out) + token * a.ot + head * a.oh;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
            if (c * 32 + lane < a.dim) orow[c * 32 + lane] = __float2bfloat16_rn(end.inv == 0.f ? 0.f : x[c] * end.c * end.inv);
        if (a.lse && lane == 0) a.lse[int64_t(token) * a.heads + head] = end.lse;
    }
}

}  // namespace cb200
