// Attention of one new token per sequence over a paged cache: flash decoding whose work is cut evenly over the CTAs,
// whatever the lengths, and joined where a cut falls inside a sequence.
//
// An item is one key-value head of one sequence with up to 8 NT of its query heads; a unit is U consecutive positions
// of it. The units of all sequences form a line, one line per head; each is cut into equal parts, one per CTA, and
// every CTA finds its part from the lengths on the device (a prefix sum over the slots), so the host reads nothing. The
// lines of the heads are cut alike and their CTAs stand side by side in the grid, so the heads of a cache row are read
// at about the same time (one line for all heads, a head after the other, read 128-byte pieces of 1 KB rows and took 8%
// longer). Within a CTA the warps take units in turn, each with its own running maximum, sum and output
// in registers, and the warps' results are merged in shared memory at the end of an item. An item that lies within one
// CTA is finished there; the others leave fp32 partial results, and the CTAs of an item's parts follow from the cut, so
// k_paged_join needs no flags or counters.
//
// Bound by HBM for long caches: keys and values are read once, and 8 query heads share them (8 multiply-adds a byte, far below what the tensor core
// could do). Short ones are bound by the latency of lengths, table, keys, values, join, each read after the other.
#pragma once

#include "mma.cuh"
#include "paged.cuh"
#include "tcgen05.cuh"

namespace cb200 {

struct PagedDecodeArgs {
    PagedArgs a;
    int blocks;      // items per key-value head
    int whole;       // one CTA per item, no cuts
    int share;       // CTAs of a cluster that share the units of a prompt's item (fp32); 1 for tokens
    int least;       // no cut leaves a CTA fewer units than this
    int q_vector;    // query rows are 16-byte aligned
    int full;        // head rows fill the padded row
    int64_t kp, kr, vp, vr;  // bytes between pages, rows
    int box;         // rows of a box of the tensor maps
    float* parts;    // [2 * CTAs][heads of an item][padded dim]
    float2* part_ml; // [2 * CTAs][heads of an item]: maximum (log2 domain) and sum
    int4* joins;     // [CTAs]: slot, item of the slot, CTAs of the line after this one, first part's number
    unsigned* error;
};

// What a token at the end of a slot sees, in units of U positions: pre units from 0, then those from main0 on, as far as
// the table goes.
template <int U> struct SeenUnits {
    int pos = -1, pre = 0, main0 = 0, units = 1;  // a slot with nothing to see has one unit with no visible key
    __device__ SeenUnits() {}
    __device__ SeenUnits(const PagedArgs& a, int slot) {
        const int last = length_of(a.lengths, slot) - 1;
        if (last >= 0) set(a, last, last);
    }
    __device__ __forceinline__ void set(const PagedArgs& a, int at, int last) {  // tokens at positions at .. last
        pos = last;
        const int low = a.window > 0 ? max(0, at - a.window + 1) : 0, top = min(last, a.width * a.page - 1);
        pre = (min(a.first, min(low, top + 1)) + U - 1) / U;
        main0 = max(low / U, pre);
        units = pre + max(0, top / U - main0 + 1);
        if (units < 1) {  // the window lies past the table
            units = 1;
            main0 = top / U;
        }
    }
    __device__ __forceinline__ int begin(int u) const { return (u < pre ? u : main0 + u - pre) * U; }
};

// The part of its line that belongs to a CTA: where it begins, and how many units it has.
template <int U> struct LinePart {
    int item, slot, u, count;  // u: unit of the slot
    SeenUnits<U> seen;
    int64_t begin, total;
    int ctas;                  // CTAs that the line is cut over
    __device__ __forceinline__ void next_slot(const PagedArgs& a) {
        u -= seen.units;
        if (++slot < a.slots) seen = SeenUnits<U>(a, slot);
    }
};

template <int U, int kWarps>
__device__ __forceinline__ LinePart<U> cut_line(const PagedDecodeArgs& p) {
    __shared__ int64_t sums[kWarps];
    __shared__ int found[2];
    const PagedArgs& a = p.a;
    const int items = a.kv * p.blocks, place = blockIdx.x / items;
    LinePart<U> part;
    part.item = blockIdx.x % items;
    part.u = part.count = 0;
    part.begin = 0;
    if (p.whole) {
        part.slot = place;
        part.seen = SeenUnits<U>(a, place);
        part.total = part.count = part.seen.units;
        part.ctas = 1;
        return part;
    }
    const int per = (a.slots + 32 * kWarps - 1) / (32 * kWarps), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int s0 = threadIdx.x * per, s1 = min(a.slots, s0 + per);
    int64_t mine = 0;
    for (int s = s0; s < s1; ++s) mine += SeenUnits<U>(a, s).units;
    int64_t upto = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    int64_t before = 0;
    part.total = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += sums[w];
        part.total += sums[w];
    }
    upto += before;
    const int64_t most = (part.total + p.least - 1) / p.least;
    part.ctas = int(gridDim.x) / items;
    if (most < part.ctas) part.ctas = int(most);
    if (place >= part.ctas) return part;
    part.begin = part.total * place / part.ctas;
    part.count = int(part.total * (place + 1) / part.ctas - part.begin);
    int64_t base = upto - mine;
    if (part.begin >= base && part.begin < upto) {
        for (int s = s0; s < s1; ++s) {
            const int units = SeenUnits<U>(a, s).units;
            if (part.begin < base + units) {
                found[0] = s;
                found[1] = int(part.begin - base);
                break;
            }
            base += units;
        }
    }
    __syncthreads();
    part.slot = found[0];
    part.u = found[1];
    part.seen = SeenUnits<U>(a, part.slot);
    return part;
}

// 16 bytes of a cache row, read once: past L1. In the order written, so that they are under way before what follows.
__device__ __forceinline__ uint4 load_word(const char* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 load_word_if(const char* p, bool ok) {
    return ok ? load_word(p) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// What is merged of one head over the warps of a CTA, over the parts of an item: weights 2^(m - M), where a part
// without a finite maximum counts only if its sum does (NaN).
__device__ __forceinline__ float part_weight(float m, float l, float top) {
    return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : fast_exp2(m - top);
}

// Final step of one head's element: o / (l + sink).
struct HeadEnd { float c, inv, lse; };
__device__ __forceinline__ HeadEnd head_end(float m, float l, float sink) {
    const float top = fmaxf(m, sink);
    const float c = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : fast_exp2(m - top);
    const float sum = l * c + (sink == -INFINITY ? 0.f : fast_exp2(sink - top));
    return HeadEnd{c, sum == 0.f ? 0.f : 1.f / sum, sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2};
}

// Running state of one warp for NT tiles of 8 heads: lane (g, t) has heads 2t and 2t + 1. o's rows are dims: with kPairs
// tile 4 d + j has dims 64 d + 8 g + 2 j (words 0, 1) and + 1 (words 2, 3), else tile j dims 16 j + g and + 8.
template <int NT, int MT> struct WarpState {
    float m[NT][2], l[NT][2], o[NT][MT][4];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int j = 0; j < MT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][j][e] = 0.f;
        }
    }
    // Scores s[kt] of 16 KT keys (log2 domain; -inf: not seen) become weights in the operand layout of the product with
    // the values. The running maximum moves only when some score exceeds it by more than 2^8, which one vote decides.
    template <int KT> __device__ __forceinline__ void weigh(const float (&s)[KT][NT][4], uint32_t (&pb)[KT][NT][2]) {
        bool grow = false;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int n = 0; n < NT; ++n)
                grow |= fmaxf(s[kt][n][0], s[kt][n][2]) > m[n][0] + 8.f || fmaxf(s[kt][n][1], s[kt][n][3]) > m[n][1] + 8.f;
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = -INFINITY;
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) x = fmaxf(x, fmaxf(s[kt][n][e], s[kt][n][e + 2]));
                    for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
                    const float top = fmaxf(m[n][e], x);
                    const float corr = m[n][e] == -INFINITY ? (l[n][e] == 0.f ? 0.f : 1.f) : fast_exp2(m[n][e] - top);
                    m[n][e] = top;
                    l[n][e] *= corr;
#pragma unroll
                    for (int j = 0; j < MT; ++j) {
                        o[n][j][e] *= corr;
                        o[n][j][e + 2] *= corr;
                    }
                }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float r0 = m[n][0] == -INFINITY ? 0.f : m[n][0], r1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                const float p0 = fast_exp2(s[kt][n][0] - r0), p1 = fast_exp2(s[kt][n][1] - r1);
                const float p2 = fast_exp2(s[kt][n][2] - r0), p3 = fast_exp2(s[kt][n][3] - r1);
                l[n][0] += p0 + p2;
                l[n][1] += p1 + p3;
                // The weights go into the product with 8 bits, as bf16 operands have; their sum keeps all of them.
                pb[kt][n][0] = transpose_8x8(pack_bf16(p0, p1));
                pb[kt][n][1] = transpose_8x8(pack_bf16(p2, p3));
            }
        }
    }
};

constexpr int kMergeDims = 64;

// The end of an item in a CTA: the warps' states are merged; a complete item is finished, of another its part is left.
template <int DP, int NT, int kWarps, bool kPairs, int MT>
__device__ __forceinline__ void end_item(const PagedDecodeArgs& p, WarpState<NT, MT>& w, int slot, int item, bool complete,
                                         int number, float* merge, float2 (*warp_ml)[8]) {
    const PagedArgs& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int kvh = item / p.blocks, head0 = (item % p.blocks) * 8 * NT;  // within the group
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
            for (int off = 4; off < 32; off <<= 1) w.l[n][e] += __shfl_xor_sync(0xffffffffu, w.l[n][e], off);
#pragma unroll
        for (int part = 0; part < DP; part += kMergeDims) {  // 64 dims at a time
            constexpr int MD = DP < kMergeDims ? DP : kMergeDims;
            __syncthreads();
            if (g == 0 && part == 0) {
                warp_ml[warp][2 * t] = make_float2(w.m[n][0], w.l[n][0]);
                warp_ml[warp][2 * t + 1] = make_float2(w.m[n][1], w.l[n][1]);
            }
            float* mine = merge + (warp * 8 + 2 * t) * MD;
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int j = part / 16; j < part / 16 + (MT < kMergeDims / 16 ? MT : kMergeDims / 16); ++j) {
                    if (kPairs) {
                        const int d = 8 * g + 2 * (j & 3);
                        if (d < MD) *reinterpret_cast<float2*>(mine + e * MD + d) = make_float2(w.o[n][j][e], w.o[n][j][e + 2]);
                    } else {
                        mine[e * MD + (j - part / 16) * 16 + g] = w.o[n][j][e];
                        mine[e * MD + (j - part / 16) * 16 + g + 8] = w.o[n][j][e + 2];
                    }
                }
            __syncthreads();
            for (int e = threadIdx.x; e < 8 * MD; e += 32 * kWarps) {
                const int r = e / MD, d = part + e % MD, in_group = head0 + n * 8 + r, head = kvh * a.group + in_group;
                if (d >= a.dim || in_group >= a.group) continue;
                float top = -INFINITY, sum = 0.f, x = 0.f;
#pragma unroll
                for (int v = 0; v < kWarps; ++v) top = fmaxf(top, warp_ml[v][r].x);
#pragma unroll
                for (int v = 0; v < kWarps; ++v) {
                    const float2 ml = warp_ml[v][r];
                    const float weight = part_weight(ml.x, ml.y, top);
                    sum += ml.y * weight;
                    x += merge[v * 8 * MD + e] * weight;
                }
                if (complete) {
                    const HeadEnd end = head_end(top, sum, sink_log2<__nv_bfloat16>(a.sinks, a.sinks_fp32, head));
                    static_cast<__nv_bfloat16*>(a.out)[slot * a.ot + head * a.oh + d] = __float2bfloat16_rn(end.inv == 0.f ? 0.f : x * end.c * end.inv);
                    if (a.lse && d == 0) a.lse[int64_t(slot) * a.heads + head] = end.lse;
                } else {
                    const int64_t at = int64_t(number) * 8 * NT + n * 8 + r;
                    p.parts[at * DP + d] = x;
                    if (d == 0) p.part_ml[at] = make_float2(top, sum);
                }
            }
        }
    }
}

// The items of a CTA's part in turn: `item(slot, seen, u0, first, last)` takes units [first, last) of the part, which are
// the slot's from u0 on, and its warps' states are merged after it.
template <int U, typename Item, typename End>
__device__ __forceinline__ void each_item(const PagedDecodeArgs& p, const LinePart<U>& part, Item&& item, End&& end) {
    int4 join = make_int4(0, 0, 0, 0);
    LinePart<U> at = part;
    for (int done = 0; done < part.count;) {
        const int take = min(part.count - done, at.seen.units - at.u);
        item(at, done, done + take);
        const bool complete = at.u == 0 && take == at.seen.units;
        const int number = 2 * blockIdx.x + (done > 0 ? 1 : 0);
        if (!complete && at.u == 0) {
            const int64_t last = part.begin + done + at.seen.units;  // one past the item's last unit
            join = make_int4(at.slot, at.item, int((last * part.ctas - 1) / part.total) - int(blockIdx.x) / (p.a.kv * p.blocks), number);
        }
        end(at, complete, number);
        done += take;
        at.u += take;
        if (at.u >= at.seen.units) at.next_slot(p.a);
    }
    if (!p.whole && threadIdx.x == 0) p.joins[blockIdx.x] = join;
}

// Warps and CTAs of an SM by the registers that a shape needs.
template <int DC, int NT> struct DecodeRegs {
    static constexpr int kWarps = 4, kCtas = DC == 4 ? 2 : DC == 2 && NT == 2 ? 3 : 4;
};

// bf16, U = 16 positions per unit, head rows of up to 32 DC values, NT tiles of 8 query heads.
//
// Scores as S^T = K Q^T with mma.m16n8k16 (16 keys x 8 heads), outputs as O^T += V^T P^T (16 dims x 8 heads): the 8
// query heads of a key-value head fill the short side of the tile, so no product is wasted on padding at 8 heads. The
// contraction of S runs over the dims in any order that K and Q share, and the columns of O may stand in any order, so
// every operand is cut such that a lane's share of a K or V row is 16 contiguous bytes: lane (g, t) of a warp loads
// dims 32 c + 8 t .. + 7 of keys g and g + 8 for S, and dims 64 d + 8 g .. + 7 of keys 2t, 2t + 1, 2t + 8, 2t + 9 for
// O. It loads them straight into registers, a unit ahead: the next unit's keys once this one's scores are done, its values
// once this one's outputs are. V's pairs of keys are put together with byte permutations, P is turned from the score
// layout into the operand layout by movmatrix.
template <int DC, int NT, bool kAligned>
__global__ void __launch_bounds__(32 * DecodeRegs<DC, NT>::kWarps, DecodeRegs<DC, NT>::kCtas)
k_paged_decode(PagedDecodeArgs p) {
    constexpr int U = 16, DB = (DC + 1) / 2, DP = 32 * DC, kWarps = DecodeRegs<DC, NT>::kWarps;
    __shared__ __align__(16) float merge[kWarps * 8 * (DP < kMergeDims ? DP : kMergeDims)];
    __shared__ float2 warp_ml[kWarps][8];
    const PagedArgs& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;" :::);
    const LinePart<U> part = cut_line<U, kWarps>(p);
    const int kvh = part.item / p.blocks, head0 = (part.item % p.blocks) * 8 * NT;  // within the group

    // This lane's share of row 0 of page 0, and the way to its other rows, in bytes.
    const char* klane = static_cast<const char*>(a.k) + (kvh * a.kh + g * a.kr + t * 8) * 2;
    const char* vlane = static_cast<const char*>(a.v) + (kvh * a.vh + 2 * t * a.vr + g * 8) * 2;
    const int64_t k8 = a.kr * 16, v1 = a.vr * 2, v8 = a.vr * 16;
    LinePart<U> next = part;  // the unit to load next, and its number in the part
    int next_index = warp;
    next.u += warp;
    const auto page_of = [&](int j, int& row) {  // page of position j (or -1), and its row there
        const int entry = int(a.by_page.div(uint32_t(j)));
        row = j - entry * a.page;
        if (entry >= a.width) return -1;
        const int id = __ldg(a.table + next.slot * a.ts + entry);
        return id < a.pages ? id : -1;
    };
    int next_id = -1, next_row = 0, next_j = 0, next_flags = 0;
    bool fast = false;           // the next unit: every row, every word
    const auto look_ahead = [&] {
        while (next.u >= next.seen.units) next.next_slot(a);
        next_j = next.seen.begin(next.u);
        if (kAligned) next_id = page_of(next_j, next_row);
    };
    uint4 kw[DC][2], vw[DB][4];  // the next unit's words of K (chunk, key g or g + 8) and V (64 dims, key)
    const auto load_keys = [&] {
        next_flags = 0;  // visibility of this lane's two keys
        if (next_index >= part.count) return;
        const int pos = next.seen.pos;
        const bool all = next_j + U - 1 <= pos && (a.window <= 0 || pos - next_j < a.window || next_j + U <= a.first);
        fast = kAligned && all && next_id >= 0 && p.full;
        if (fast) {
            const char* k = klane + p.kp * next_id + p.kr * next_row;
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                kw[c][0] = load_word(k + c * 64);
                kw[c][1] = load_word(k + k8 + c * 64);
            }
            next_flags = 3;
        } else {  // rows that are not seen, and words past the head's row, are zeros
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int j = next_j + g + 8 * h;
                int row = next_row + 8 * h, id = next_id;
                if (!kAligned) id = page_of(j, row), row -= g;
                const bool ok = id >= 0 && (all || sees(pos, j, a.window, a.first));
                next_flags |= int(ok) << h;
                const char* k = klane + p.kp * id + p.kr * row;
#pragma unroll
                for (int c = 0; c < DC; ++c) kw[c][h] = load_word_if(k + c * 64, ok && c * 32 + t * 8 < a.dim);
            }
        }
    };
    const auto load_values = [&] {  // of the unit whose keys were loaded last; then the next unit is looked up
        if (next_index >= part.count) return;
        const int pos = next.seen.pos;
        if (fast) {
            const char* v = vlane + p.vp * next_id + p.vr * next_row;
            const bool ok = DP >= 64 || g * 8 < DP;  // a row of 32 values ends after the words of half of the lanes
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                vw[d][0] = load_word_if(v + d * 128, ok);
                vw[d][1] = load_word_if(v + v1 + d * 128, ok);
                vw[d][2] = load_word_if(v + v8 + d * 128, ok);
                vw[d][3] = load_word_if(v + v8 + v1 + d * 128, ok);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = (e & 1) + (e >> 1) * 8, j = next_j + 2 * t + r;
                int row = next_row + r, id = next_id;
                if (!kAligned) id = page_of(j, row), row -= 2 * t;
                const bool ok = id >= 0 && sees(pos, j, a.window, a.first);
                const char* v = vlane + p.vp * id + p.vr * row;
#pragma unroll
                for (int d = 0; d < DB; ++d) vw[d][e] = load_word_if(v + d * 128, ok && d * 64 + g * 8 < a.dim);
            }
        }
        next_index += kWarps;
        next.u += kWarps;
        if (next_index < part.count) look_ahead();
    };
    if (next_index < part.count) look_ahead();
    load_keys();
    load_values();

    WarpState<NT, DB * 4> w;
    each_item<U>(p, part, [&](const LinePart<U>& at, int first, int last) {
        uint4 q[NT][DC];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                const int head = head0 + n * 8 + g, d = c * 32 + t * 8;
                q[n][c] = make_uint4(0, 0, 0, 0);
                if (head < a.group && d < a.dim) {
                    const auto* row = static_cast<const __nv_bfloat16*>(a.q) + at.slot * a.qt + (int64_t(kvh) * a.group + head) * a.qh + d;
                    if (p.q_vector) q[n][c] = __ldg(reinterpret_cast<const uint4*>(row));
                    else {
                        const auto* h = reinterpret_cast<const uint16_t*>(row);
                        q[n][c] = make_uint4(h[0] | uint32_t(h[1]) << 16, h[2] | uint32_t(h[3]) << 16,
                                             h[4] | uint32_t(h[5]) << 16, h[6] | uint32_t(h[7]) << 16);
                    }
                }
            }
        w.clear();
        for (int k = first + (warp - first % kWarps + kWarps) % kWarps; k < last; k += kWarps) {
            const int vis = next_flags;
            float s[1][NT][4], half[NT][4];  // two chains of products
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[0][n][e] = half[n][e] = 0.f;
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                const uint4 ka = kw[c][0], kb = kw[c][1];
                const uint32_t a0[4] = {ka.x, kb.x, ka.y, kb.y}, a1[4] = {ka.z, kb.z, ka.w, kb.w};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma_bf16(s[0][n], a0, q[n][c].x, q[n][c].y);
                    mma_bf16(half[n], a1, q[n][c].z, q[n][c].w);
                }
            }
            load_keys();
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s[0][n][e] = (vis >> (e >> 1)) & 1 ? (s[0][n][e] + half[n][e]) * a.scale_log2 : -INFINITY;
            uint32_t pb[1][NT][2];
            w.template weigh<1>(s, pb);
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const auto& v = vw[d];
                const auto word = [](const uint4& x, int j) { return j == 0 ? x.x : j == 1 ? x.y : j == 2 ? x.z : x.w; };
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // dims 64 d + 8 g + 2 j (rows g) and + 1 (rows g + 8)
                    const uint32_t f[4] = {__byte_perm(word(v[0], j), word(v[1], j), 0x5410), __byte_perm(word(v[0], j), word(v[1], j), 0x7632),
                                           __byte_perm(word(v[2], j), word(v[3], j), 0x5410), __byte_perm(word(v[2], j), word(v[3], j), 0x7632)};
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_bf16(w.o[n][d * 4 + j], f, pb[0][n][0], pb[0][n][1]);
                }
            }
            load_values();
        }
    }, [&](const LinePart<U>& at, bool complete, int number) {
        end_item<DP, NT, kWarps, true>(p, w, at.slot, at.item, complete, number, merge, warp_ml);
    });
}

// The same from a ring in shared memory that the TMA engine fills, for head rows of 64 or 128 values and pages of a
// multiple of 16 rows: U positions of K and of V per stage, 128-byte swizzle, read with ldmatrix (transposed for V).
// Every warp has its own ring and issues its own loads, kStages ahead, so there is no barrier between warps, and two to
// three times as many bytes are under way as registers could hold: bound by HBM. 128 sequences of 1,024-4,096 positions
// (64/8 heads of 64): 115 us of kernel, 120 with its launches and the join, 5.6 TB/s (k_paged_decode 142); two of 40,001 and
// 131,071 (32/8 heads of 128): 139 us, 6.05 TB/s. A ring of cp.async took 194 for the first. Eight warps on an SM are enough: sixteen with half the positions a stage took as long.
template <int DC> struct DecodeRing {
    static constexpr int U = DC == 2 ? 32 : 16, kWarps = 4, kStages = 3, kTile = U * 64 * DC, kStage = 2 * kTile;
    static constexpr int kSmem = 1024 + kWarps * (kStages * kStage + 8 * kMergeDims * 4);
};

// Box {64 values, 1 head, rows, 1 page} of a pool.
__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, int d, int head, int row, int page,
                                              uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
            "r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(d), "r"(head), "r"(row), "r"(page), "r"(smem_addr(bar))
        : "memory");
}

template <int DC, int NT>
__global__ void __launch_bounds__(32 * DecodeRing<DC>::kWarps, 2)
k_paged_decode_tma(PagedDecodeArgs p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using Ring = DecodeRing<DC>;
    constexpr int U = Ring::U, KT = U / 16, MT = 2 * DC, DP = 32 * DC, kWarps = Ring::kWarps, kStages = Ring::kStages;
    constexpr int kHalf = U * 128;  // bytes of 64 values of U rows
    extern __shared__ uint8_t dec_raw[];
    __shared__ uint64_t full[kWarps][kStages];
    __shared__ float2 warp_ml[kWarps][8];
    const PagedArgs& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t base = (smem_addr(dec_raw) + 1023) & ~1023u;
    const uint32_t ring = base + warp * kStages * Ring::kStage;
    float* merge = reinterpret_cast<float*>(dec_raw + (base - smem_addr(dec_raw)) + kWarps * kStages * Ring::kStage);
    asm volatile("griddepcontrol.launch_dependents;" :::);
    if (lane == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(&full[warp][s], 1);
        fence_barrier_init();
        if (warp == 0) {
            prefetch_tensormap(&kmap);
            prefetch_tensormap(&vmap);
        }
    }
    __syncwarp();
    const LinePart<U> part = cut_line<U, kWarps>(p);
    const int kvh = part.item / p.blocks, head0 = (part.item % p.blocks) * 8 * NT;  // within the group

    // ---- load side: this warp's units in turn
    LinePart<U> next = part;
    int next_index = warp, issued = 0;
    uint32_t missing = 0;   // per unit under way, the last one lowest: two bits, a page that is not there
    int id[KT], row[KT];    // of the next unit's boxes (of 16 rows; those of 32 rows use the first)
    next.u += warp;
    const auto look_ahead = [&] {
        while (next.u >= next.seen.units) next.next_slot(a);
#pragma unroll
        for (int i = 0; i < KT; ++i) {
            if (i && p.box == U) break;
            const int j = next.seen.begin(next.u) + 16 * i, entry = int(a.by_page.div(uint32_t(j)));
            row[i] = j - entry * a.page;
            id[i] = entry < a.width ? __ldg(a.table + next.slot * a.ts + entry) : -1;
            if (id[i] < 0 || id[i] >= a.pages) id[i] = a.pages;  // beyond the map: zeros
        }
    };
    const auto issue = [&] {
        missing <<= 2;
        if (next_index >= part.count) return;
        const int stage = issued % kStages;
        if (lane == 0) {
            uint64_t* bar = &full[warp][stage];
            const uint32_t dst = ring + stage * Ring::kStage;
            mbar_arrive_expect_tx(bar, Ring::kStage);
#pragma unroll
            for (int i = 0; i < KT; ++i) {
                if (i && p.box == U) break;
#pragma unroll
                for (int d = 0; d < DC / 2; ++d) {
                    tma_load_page(dst + d * kHalf + i * 2048, &kmap, d * 64, kvh, row[i], id[i], bar);
                    tma_load_page(dst + Ring::kTile + d * kHalf + i * 2048, &vmap, d * 64, kvh, row[i], id[i], bar);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < KT; ++i) missing |= uint32_t(id[p.box == U ? 0 : i] >= a.pages) << i;
        ++issued;
        next_index += kWarps;
        next.u += kWarps;
        if (next_index < part.count) look_ahead();
    };
    if (next_index < part.count) look_ahead();
#pragma unroll
    for (int s = 0; s < kStages; ++s) issue();

    // ---- use side
    int used = 0;
    bool alive = true;
    // ldmatrix rows: K's 16 keys x 16 dims as the A operand; V's transposed, 16 dims x 16 keys.
    const uint32_t krow = uint32_t((lane & 7) + ((lane >> 3) & 1) * 8), kcol = uint32_t(lane >> 4);
    const uint32_t vrow = uint32_t((lane & 7) + (lane >> 4) * 8), vcol = uint32_t((lane >> 3) & 1);
    WarpState<NT, MT> w;
    each_item<U>(p, part, [&](const LinePart<U>& at, int first, int last) {
        uint32_t q[NT][MT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int head = head0 + n * 8 + g;
            const auto* qrow = reinterpret_cast<const uint16_t*>(a.q) + at.slot * a.qt + (int64_t(kvh) * a.group + head) * a.qh + 2 * t;
#pragma unroll
            for (int c = 0; c < MT; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint16_t* x = qrow + c * 16 + h * 8;
                    q[n][c][h] = head >= a.group ? 0 : p.q_vector ? __ldg(reinterpret_cast<const uint32_t*>(x)) : x[0] | uint32_t(x[1]) << 16;
                }
        }
        w.clear();
        for (int k = first + (warp - first % kWarps + kWarps) % kWarps; k < last; k += kWarps) {
            const int stage = used % kStages, j0 = at.seen.begin(at.u + k - first), pos = at.seen.pos;
            const uint32_t gone = missing >> (2 * (kStages - 1));
            if (alive) alive = mbar_wait(&full[warp][stage], (used / kStages) & 1, p.error);
            ++used;
            const uint32_t ks = ring + stage * Ring::kStage, vs = ks + Ring::kTile;
            float s[KT][NT][4];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                float half[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[kt][n][e] = half[n][e] = 0.f;
#pragma unroll
                for (int c = 0; c < MT; ++c) {
                    uint32_t f[4];
                    ldsm_x4(f, ks + (c >> 2) * kHalf + (kt * 16 + krow) * 128 + ((((c & 3) * 2 + kcol) ^ (krow & 7)) << 4));
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_bf16(c & 1 ? half[n] : s[kt][n], f, q[n][c][0], q[n][c][1]);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[kt][n][e] = (s[kt][n][e] + half[n][e]) * a.scale_log2;
            }
            if (!(j0 + U - 1 <= pos && (a.window <= 0 || pos - j0 < a.window || j0 + U <= a.first)) || (gone & 3)) {
                // Keys that are not seen: no score, and zeros for values (what lies there may not be finite).
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if ((gone >> kt & 1) || !sees(pos, j0 + kt * 16 + g + 8 * (e >> 1), a.window, a.first)) s[kt][n][e] = -INFINITY;
                if (lane < U && !sees(pos, j0 + lane, a.window, a.first))
#pragma unroll
                    for (int c = 0; c < DC * 4; ++c)
                        asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(vs + (c >> 3) * kHalf + lane * 128 + (c & 7) * 16), "r"(0) : "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            uint32_t pb[KT][NT][2];
            w.template weigh<KT>(s, pb);
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int c = 0; c < MT; ++c) {
                    uint32_t f[4];
                    ldsm_x4_t(f, vs + (c >> 2) * kHalf + (kt * 16 + vrow) * 128 + ((((c & 3) * 2 + vcol) ^ (vrow & 7)) << 4));
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_bf16(w.o[n][c], f, pb[kt][n][0], pb[kt][n][1]);
                }
            __syncwarp();
            if (alive) issue();
        }
    }, [&](const LinePart<U>& at, bool complete, int number) {
        end_item<DP, NT, kWarps, false>(p, w, at.slot, at.item, complete, number, merge, warp_ml);
    });
    // After a wait that gave up: the copies still under way end (or are given up too) before the memory is left.
    if (!alive)
        for (; used < issued; ++used)
            if (!mbar_wait(&full[warp][used % kStages], (used / kStages) & 1, p.error)) break;
}

// Joins the parts of the item that begins in CTA blockIdx.x's part of its line and goes on after it (if there is one),
// in the order of the parts: one CTA for one query head of it (blockIdx.y) whose 8 warps share the parts, or, with
// kWarp, one CTA for 8 heads and a warp for each.
template <typename T, int DP, bool kWarp> __global__ void __launch_bounds__(256) k_paged_join(PagedDecodeArgs p, int item_heads) {
    __shared__ float sums[kWarp ? 1 : 8][DP];
    __shared__ float totals[8];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 join = p.joins[blockIdx.x];
    const PagedArgs& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r = kWarp ? blockIdx.y * 8 + warp : blockIdx.y, items = a.kv * p.blocks, n = join.z + 1;
    const int in_group = join.y % p.blocks * item_heads + r, head = join.y / p.blocks * a.group + in_group;
    if (join.z == 0 || in_group >= a.group) return;
    const auto part = [&](int i) { return int64_t(i == 0 ? join.w : 2 * (int(blockIdx.x) + i * items)) * item_heads + r; };
    float top = -INFINITY, sum = 0.f, x[DP / 32] = {};
    for (int i = lane; i < n; i += 32) top = fmaxf(top, p.part_ml[part(i)].x);
    top = warp_max(top);
    for (int i = kWarp ? 0 : warp; i < n; i += kWarp ? 1 : 8) {
        const float2 ml = p.part_ml[part(i)];
        const float w = part_weight(ml.x, ml.y, top);
        sum += ml.y * w;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c)
            if (c * 32 + lane < a.dim) x[c] += p.parts[part(i) * DP + c * 32 + lane] * w;
    }
    if (!kWarp) {
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) sums[warp][c * 32 + lane] = x[c];
        if (lane == 0) totals[warp] = sum;
        __syncthreads();
        if (warp) return;
        sum = 0.f;
        for (int v = 0; v < 8; ++v) sum += totals[v];
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
            x[c] = 0.f;
            for (int v = 0; v < 8; ++v) x[c] += sums[v][c * 32 + lane];
        }
    }
    const HeadEnd end_of = head_end(top, sum, sink_log2<T>(a.sinks, a.sinks_fp32, head));
#pragma unroll
    for (int c = 0; c < DP / 32; ++c)
        if (c * 32 + lane < a.dim)
            Store<T>::store(static_cast<T*>(a.out) + join.x * a.ot + head * a.oh + c * 32 + lane,
                            end_of.inv == 0.f ? 0.f : x[c] * end_of.c * end_of.inv);
    if (a.lse && lane == 0) a.lse[int64_t(join.x) * a.heads + head] = end_of.lse;
}

}  // namespace cb200
