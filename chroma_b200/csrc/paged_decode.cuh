// Attention of one new token per sequence over a paged cache: flash decoding whose work is cut evenly over the CTAs,
// whatever the lengths, and joined where a cut falls inside a sequence.
//
// An item is one key-value head of one sequence with up to 8 NT of its query heads; a unit is U consecutive positions
// of it. All units of all items form one line, cut into equal parts, one per CTA; every CTA finds its part from the
// lengths on the device (a prefix sum over the slots), so the host reads nothing. Within a CTA the 8 warps take units
// in turn, each with its own running maximum, sum and output in registers, and the warps' results are merged in shared
// memory at the end of an item. An item that lies within one CTA is finished there; the others leave fp32 partial
// results, and the CTA numbers of an item's parts follow from the cut, so k_paged_join needs no flags or counters.
#pragma once

#include "paged.cuh"
#include "tma.cuh"

namespace cb200 {

constexpr int kDecWarps = 8, kDecThreads = 32 * kDecWarps;

struct PagedDecodeArgs {
    PagedArgs a;
    int blocks;      // head blocks per key-value head
    int whole;       // one CTA per item, no cuts
    int least;       // no cut leaves a CTA fewer units than this
    int q_vector;    // query rows are 16-byte aligned
    int full;        // head rows fill the padded row
    int64_t kp, kr, vp, vr;  // bytes between pages, rows
    float* parts;    // [2 * CTAs][heads of a block][padded dim]
    float2* part_ml; // [2 * CTAs][heads of a block]: maximum (log2 domain) and sum
    int4* joins;     // [CTAs]: slot, item of the slot, CTAs after this one, first part's number
};

// What a token at the end of a slot sees, in units of U positions: pre units from 0, then those from main0 on.
template <int U> struct SeenUnits {
    int pos = -1, pre = 0, main0 = 0, units = 1;  // a slot with nothing to see has one unit with no visible key
    __device__ SeenUnits() {}
    __device__ SeenUnits(const PagedArgs& a, int slot) {
        pos = held_rows(a.lengths, slot, a.width, a.page) - 1;
        if (pos < 0) return;
        const int low = a.window > 0 ? max(0, pos - a.window + 1) : 0;
        pre = (min(a.first, low) + U - 1) / U;
        main0 = max(low / U, pre);
        units = pre + pos / U - main0 + 1;
        if (units < 1) units = 1;
    }
    __device__ __forceinline__ int begin(int u) const { return (u < pre ? u : main0 + u - pre) * U; }
};

// A place in the line of units.
template <int U> struct UnitCursor {
    int slot, item, u;
    SeenUnits<U> seen;
    __device__ void normalise(const PagedArgs& a, int items) {
        while (u >= seen.units) {
            u -= seen.units;
            if (++item == items) {
                item = 0;
                if (++slot < a.slots) seen = SeenUnits<U>(a, slot);
                else {
                    u = 0;
                    return;
                }
            }
        }
    }
};

// The part of the line that belongs to this CTA: where it begins, and how many units it has.
template <int U> struct CtaPart {
    int64_t begin, count, total;
    int ctas;
};

template <int U>
__device__ __forceinline__ CtaPart<U> cut_line(const PagedDecodeArgs& p, int items, UnitCursor<U>& at) {
    __shared__ int64_t sums[kDecWarps];
    __shared__ int found[3];
    const PagedArgs& a = p.a;
    CtaPart<U> part;
    if (p.whole) {
        at.slot = blockIdx.x / items;
        at.item = blockIdx.x % items;
        at.u = 0;
        at.seen = SeenUnits<U>(a, at.slot);
        part.begin = 0;
        part.count = part.total = at.seen.units;
        part.ctas = 1;
        return part;
    }
    const int per = (a.slots + kDecThreads - 1) / kDecThreads, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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
    int64_t before = 0, all = 0;
    for (int w = 0; w < kDecWarps; ++w) {
        if (w < warp) before += sums[w];
        all += sums[w];
    }
    upto += before;
    part.total = all * items;
    const int64_t most = (part.total + p.least - 1) / p.least;
    part.ctas = int(most < gridDim.x ? most : gridDim.x);
    if (int(blockIdx.x) >= part.ctas) {
        part.begin = part.count = 0;
        return part;
    }
    part.begin = part.total * blockIdx.x / part.ctas;
    part.count = part.total * (blockIdx.x + 1) / part.ctas - part.begin;
    int64_t base = (upto - mine) * items;
    if (part.begin >= base && part.begin < upto * items) {
        for (int s = s0; s < s1; ++s) {
            const int units = SeenUnits<U>(a, s).units;
            if (part.begin < base + int64_t(units) * items) {
                found[0] = s;
                found[1] = int((part.begin - base) / units);
                found[2] = int((part.begin - base) % units);
                break;
            }
            base += int64_t(units) * items;
        }
    }
    __syncthreads();
    at.slot = found[0];
    at.item = found[1];
    at.u = found[2];
    at.seen = SeenUnits<U>(a, at.slot);
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
__device__ __forceinline__ float exp2_sfu(float x) {  // 2^-inf = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// D (16 x 8, fp32) += A (16 x 16) B (16 x 8), bf16.
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// What is merged of one head over the warps of a CTA, over the parts of an item: weights 2^(m - M), where a part
// without a finite maximum counts only if its sum does (NaN).
__device__ __forceinline__ float part_weight(float m, float l, float top) {
    return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2_sfu(m - top);
}

// Final step of one head's element: o / (l + sink).
struct HeadEnd { float c, inv, lse; };
__device__ __forceinline__ HeadEnd head_end(float m, float l, float sink) {
    const float top = fmaxf(m, sink);
    const float c = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2_sfu(m - top);
    const float sum = l * c + (sink == -INFINITY ? 0.f : exp2_sfu(sink - top));
    return HeadEnd{c, sum == 0.f ? 0.f : 1.f / sum, sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2};
}

// bf16, U = 16 positions per unit, head rows of up to 32 DC values, NT tiles of 8 query heads.
//
// Scores as S^T = K Q^T with mma.m16n8k16 (16 keys x 8 heads), outputs as O^T += V^T P^T (16 dims x 8 heads): the 8
// query heads of a key-value head fill the short side of the tile, so no product is wasted on padding at 8 heads. The
// contraction of S runs over the dims in any order that K and Q share, and the columns of O may stand in any order, so
// every operand is cut such that a lane's share of a K or V row is 16 contiguous bytes: lane (g, t) of a warp loads
// dims 32 c + 8 t .. + 7 of keys g and g + 8 for S, and dims 64 d + 8 g .. + 7 of keys 2t, 2t + 1, 2t + 8, 2t + 9 for
// O. It copies them with cp.async into slots of shared memory that only it reads, a ring of stages ahead, so the ring
// needs no barrier at all. V's pairs of keys are put together with byte permutations, P is turned from the score
// layout into the operand layout by movmatrix.
//
// The running maximum moves only when some score exceeds it by more than 2^8, which one vote decides; sums and
// products stay within 2^8 of their exact scale, and nothing is exchanged between lanes otherwise.
template <int DC, int NT, bool kAligned>
__global__ void __launch_bounds__(kDecThreads, DC == 4 ? 1 : 2) k_paged_decode(PagedDecodeArgs p) {
    constexpr int U = 16, DB = (DC + 1) / 2, DP = 32 * DC;
    __shared__ __align__(16) float merge[kDecWarps * 8 * DP];
    __shared__ float2 warp_ml[kDecWarps][8];
    const PagedArgs& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int items = a.kv * p.blocks;
    asm volatile("griddepcontrol.launch_dependents;" :::);

    UnitCursor<U> at;
    const CtaPart<U> part = cut_line<U>(p, items, at);
    int4 join = make_int4(0, 0, 0, 0);
    const int count = int(part.count);
    if (count == 0) {
        if (!p.whole && threadIdx.x == 0) p.joins[blockIdx.x] = join;
        return;
    }

    // ---- load side: this warp's units in turn, one ahead
    UnitCursor<U> next = at;
    int next_index = warp, next_id = -1, next_row = 0;
    next.u += warp;
    next.normalise(a, items);
    // Byte addresses of this lane's share of row 0 of page 0 for the item's key-value head, and its other rows.
    const char *klane, *vlane;
    const int64_t k8 = a.kr * 16, v1 = a.vr * 2, v8 = a.vr * 16;
    const auto enter_item = [&] {
        const int64_t kvh = next.item / p.blocks;
        klane = static_cast<const char*>(a.k) + (kvh * a.kh + g * a.kr + t * 8) * 2;
        vlane = static_cast<const char*>(a.v) + (kvh * a.vh + 2 * t * a.vr + g * 8) * 2;
    };
    const auto page_of = [&](int j, int& row) {  // page of position j of the next unit's slot (or -1), and its row
        const int entry = int(a.by_page.div(uint32_t(j)));
        row = j - entry * a.page;
        if (entry >= a.width) return -1;
        const int id = __ldg(a.table + next.slot * a.ts + entry);
        return id < a.pages ? id : -1;
    };
    const auto fetch_id = [&] {  // a unit ahead of its use
        if (kAligned) next_id = page_of(next.seen.begin(next.u), next_row);
    };
    if (next_index < count) {
        enter_item();
        fetch_id();
    }
    uint4 kw[DC][2], vw[DB][4];  // the next unit's words of K (chunk, key g or g + 8) and V (64 dims, key)
    int next_flags = 0;          // visibility of this lane's two keys
    bool fast = false;           // every row, every word
    const auto load_keys = [&] {
        next_flags = 0;
        if (next_index >= count) return;
        const int j0 = next.seen.begin(next.u), pos = next.seen.pos;
        const bool all = j0 + U - 1 <= pos && (a.window <= 0 || pos - j0 < a.window || j0 + U <= a.first);
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
                const int j = j0 + g + 8 * h;
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
    // The values of the unit whose keys were loaded last; then the cursor moves on.
    const auto load_values = [&] {
        if (next_index >= count) return;
        if (fast) {
            const char* v = vlane + p.vp * next_id + p.vr * next_row;
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                vw[d][0] = load_word(v + d * 128);
                vw[d][1] = load_word(v + v1 + d * 128);
                vw[d][2] = load_word(v + v8 + d * 128);
                vw[d][3] = load_word(v + v8 + v1 + d * 128);
            }
        } else {
            const int j0 = next.seen.begin(next.u), pos = next.seen.pos;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = (e & 1) + (e >> 1) * 8, j = j0 + 2 * t + r;
                int row = next_row + r, id = next_id;
                if (!kAligned) id = page_of(j, row), row -= 2 * t;
                const bool ok = id >= 0 && sees(pos, j, a.window, a.first);
                const char* v = vlane + p.vp * id + p.vr * row;
#pragma unroll
                for (int d = 0; d < DB; ++d) vw[d][e] = load_word_if(v + d * 128, ok && d * 64 + g * 8 < a.dim);
            }
        }
        next_index += kDecWarps;
        next.u += kDecWarps;
        if (next_index < count) {
            if (next.u >= next.seen.units) {
                next.normalise(a, items);
                enter_item();
            }
            fetch_id();
        }
    };
    load_keys();
    load_values();

    // ---- use side, item by item
    int done = 0;
    int slot = at.slot, item = at.item, u0 = at.u;
    SeenUnits<U> seen = at.seen;
    while (done < count) {
        const int take = min(count - done, seen.units - u0);
        const int kvh = item / p.blocks, head0 = (item % p.blocks) * 8 * NT;  // within the group
        uint4 q[NT][DC];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                const int head = head0 + n * 8 + g, d = c * 32 + t * 8;
                q[n][c] = make_uint4(0, 0, 0, 0);
                if (head < a.group && d < a.dim) {
                    const auto* row = static_cast<const __nv_bfloat16*>(a.q) + slot * a.qt + (int64_t(kvh) * a.group + head) * a.qh + d;
                    if (p.q_vector) q[n][c] = __ldg(reinterpret_cast<const uint4*>(row));
                    else {
                        const auto* h = reinterpret_cast<const uint16_t*>(row);
                        q[n][c] = make_uint4(h[0] | uint32_t(h[1]) << 16, h[2] | uint32_t(h[3]) << 16,
                                             h[4] | uint32_t(h[5]) << 16, h[6] | uint32_t(h[7]) << 16);
                    }
                }
            }
        float m[NT][2], l[NT][2], o[NT][DB * 4][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int j = 0; j < DB * 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][j][e] = 0.f;
        }
        const int end = done + take;
        for (int k = done + (unsigned(warp - done) % kDecWarps); k < end; k += kDecWarps) {
            const int vis = next_flags;
            float s[NT][4], half[NT][4];  // two chains of products
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = half[n][e] = 0.f;
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                const uint4 ka = kw[c][0], kb = kw[c][1];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma_16816(s[n], ka.x, kb.x, ka.y, kb.y, q[n][c].x, q[n][c].y);
                    mma_16816(half[n], ka.z, kb.z, ka.w, kb.w, q[n][c].z, q[n][c].w);
                }
            }
            load_keys();
            bool grow = false;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[n][e] = (s[n][e] + half[n][e]) * a.scale_log2;
                    if (!((vis >> (e >> 1)) & 1)) s[n][e] = -INFINITY;
                }
                grow |= fmaxf(s[n][0], s[n][2]) > m[n][0] + 8.f || fmaxf(s[n][1], s[n][3]) > m[n][1] + 8.f;
            }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = fmaxf(s[n][e], s[n][e + 2]);
                        for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
                        const float top = fmaxf(m[n][e], x);
                        const float corr = m[n][e] == -INFINITY ? (l[n][e] == 0.f ? 0.f : 1.f) : exp2_sfu(m[n][e] - top);
                        m[n][e] = top;
                        l[n][e] *= corr;
#pragma unroll
                        for (int j = 0; j < DB * 4; ++j) {
                            o[n][j][e] *= corr;
                            o[n][j][e + 2] *= corr;
                        }
                    }
            }
            uint32_t pb[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float r0 = m[n][0] == -INFINITY ? 0.f : m[n][0], r1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
                const float p0 = exp2_sfu(s[n][0] - r0), p1 = exp2_sfu(s[n][1] - r1);
                const float p2 = exp2_sfu(s[n][2] - r0), p3 = exp2_sfu(s[n][3] - r1);
                l[n][0] += p0 + p2;
                l[n][1] += p1 + p3;
                // The weights go into the product with 8 bits, as bf16 operands have; their sum keeps all of them.
                pb[n][0] = transpose_8x8(bf16_pair(p0, p1));
                pb[n][1] = transpose_8x8(bf16_pair(p2, p3));
            }
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const auto& v = vw[d];
                const auto word = [](const uint4& x, int j) { return j == 0 ? x.x : j == 1 ? x.y : j == 2 ? x.z : x.w; };
#pragma unroll
                for (int j = 0; j < 4; ++j) {  // dims 64 d + 8 g + 2 j (rows g) and + 1 (rows g + 8)
                    const uint32_t a0 = __byte_perm(word(v[0], j), word(v[1], j), 0x5410);
                    const uint32_t a1 = __byte_perm(word(v[0], j), word(v[1], j), 0x7632);
                    const uint32_t a2 = __byte_perm(word(v[2], j), word(v[3], j), 0x5410);
                    const uint32_t a3 = __byte_perm(word(v[2], j), word(v[3], j), 0x7632);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816(o[n][d * 4 + j], a0, a1, a2, a3, pb[n][0], pb[n][1]);
                }
            }
            load_values();
        }
        // ---- the item's end: merge the warps, then finish it or leave its part
        const bool complete = u0 == 0 && take == seen.units;
        const int number = 2 * blockIdx.x + (done > 0 ? 1 : 0);
        if (!complete && u0 == 0) {
            const int64_t last = part.begin + done + seen.units;  // one past the item's last unit
            join = make_int4(slot, item, int((last * part.ctas - 1) / part.total) - int(blockIdx.x), number);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
                for (int off = 4; off < 32; off <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], off);
            __syncthreads();
            if (g == 0) {
                warp_ml[warp][2 * t] = make_float2(m[n][0], l[n][0]);
                warp_ml[warp][2 * t + 1] = make_float2(m[n][1], l[n][1]);
            }
#pragma unroll
            for (int d = 0; d < DB; ++d)
                if (d * 64 + g * 8 < DP)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float4* row = reinterpret_cast<float4*>(merge + (warp * 8 + 2 * t + e) * DP + d * 64 + g * 8);
                        row[0] = make_float4(o[n][d * 4][e], o[n][d * 4][e + 2], o[n][d * 4 + 1][e], o[n][d * 4 + 1][e + 2]);
                        row[1] = make_float4(o[n][d * 4 + 2][e], o[n][d * 4 + 2][e + 2], o[n][d * 4 + 3][e], o[n][d * 4 + 3][e + 2]);
                    }
            __syncthreads();
            for (int e = threadIdx.x; e < 8 * DP; e += kDecThreads) {
                const int r = e / DP, d = e % DP, in_group = head0 + n * 8 + r;
                if (d >= a.dim || in_group >= a.group) continue;
                float top = -INFINITY, sum = 0.f, x = 0.f;
#pragma unroll
                for (int w = 0; w < kDecWarps; ++w) top = fmaxf(top, warp_ml[w][r].x);
#pragma unroll
                for (int w = 0; w < kDecWarps; ++w) {
                    const float2 ml = warp_ml[w][r];
                    const float weight = part_weight(ml.x, ml.y, top);
                    sum += ml.y * weight;
                    x += merge[(w * 8 + r) * DP + d] * weight;
                }
                if (complete) {
                    const int head = kvh * a.group + in_group;
                    const HeadEnd end_of = head_end(top, sum, sink_log2<__nv_bfloat16>(a.sinks, a.sinks_fp32, head));
                    static_cast<__nv_bfloat16*>(a.out)[slot * a.ot + head * a.oh + d] = __float2bfloat16_rn(end_of.inv == 0.f ? 0.f : x * end_of.c * end_of.inv);
                    if (a.lse && d == 0) a.lse[int64_t(slot) * a.heads + head] = end_of.lse;
                } else {
                    p.parts[(int64_t(number) * 8 * NT + n * 8 + r) * DP + d] = x;
                    if (d == 0) p.part_ml[int64_t(number) * 8 * NT + n * 8 + r] = make_float2(top, sum);
                }
            }
        }
        done += take;
        u0 = 0;
        if (++item == items) {
            item = 0;
            if (++slot < a.slots) seen = SeenUnits<U>(a, slot);
        }
    }
    if (!p.whole && threadIdx.x == 0) p.joins[blockIdx.x] = join;
}

// Joins the parts of the item that begins in CTA blockIdx.x's part of the line and goes on after it (if there is one),
// for head blockIdx.y of its block, in the order of the parts.
template <typename T, int DP> __global__ void __launch_bounds__(128) k_paged_join(PagedDecodeArgs p, int block_heads) {
    __shared__ float weights[1024], red[4], sums[4][DP];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 join = p.joins[blockIdx.x];
    const PagedArgs& a = p.a;
    const int in_group = (join.y % p.blocks) * block_heads + blockIdx.y;
    if (join.z == 0 || in_group >= a.group) return;
    const int n = join.z + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = (join.y / p.blocks) * a.group + in_group;
    const auto number = [&](int i) { return i == 0 ? join.w : 2 * (int(blockIdx.x) + i); };
    const auto ml = [&](int i) { return p.part_ml[int64_t(number(i)) * block_heads + blockIdx.y]; };
    float top = -INFINITY;
    for (int i = threadIdx.x; i < n; i += 128) top = fmaxf(top, ml(i).x);
    top = warp_max(top);
    if (lane == 0) red[warp] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float sum = 0.f;
    for (int i = threadIdx.x; i < n; i += 128) {
        const float2 v = ml(i);
        weights[i] = part_weight(v.x, v.y, top);
        sum += v.y * weights[i];
    }
    sum = warp_sum(sum);
    __syncthreads();
    if (lane == 0) red[warp] = sum;
    float x[DP / 32] = {};
    for (int i = warp; i < n; i += 4) {
        const float w = weights[i];
        const float* part = p.parts + (int64_t(number(i)) * block_heads + blockIdx.y) * DP;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c)
            if (c * 32 + lane < a.dim) x[c] += part[c * 32 + lane] * w;
    }
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) sums[warp][c * 32 + lane] = x[c];
    __syncthreads();
    sum = (red[0] + red[1]) + (red[2] + red[3]);
    const HeadEnd end_of = head_end(top, sum, sink_log2<T>(a.sinks, a.sinks_fp32, head));
    for (int d = threadIdx.x; d < a.dim; d += 128) {
        const float v = (sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d]);
        Store<T>::store(static_cast<T*>(a.out) + join.x * a.ot + head * a.oh + d, end_of.inv == 0.f ? 0.f : v * end_of.c * end_of.inv);
    }
    if (a.lse && threadIdx.x == 0) a.lse[int64_t(join.x) * a.heads + head] = end_of.lse;
}

}  // namespace cb200
