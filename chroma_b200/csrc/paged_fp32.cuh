// fp32 attention over a paged cache, single tokens and prompts, on the FMA pipe (tensor-core products of fp32 operands would
// keep 11 or 8 of their 24 bits).
//
// An item is up to 8 rows that share a key-value head: query heads of one token, or, where a key-value head has fewer than
// 8 of them, of several consecutive tokens. Units of 32 positions are dealt to the 8 warps of a CTA. A lane has one key of
// the unit: it walks the key's row in 16-byte words and multiplies each with the same words of the 8 query rows, which all
// lanes read from the same place of shared memory, so a score needs no exchange between lanes. The values are read with a
// row spread over `kWords` lanes, weights come from the lane of their key by shuffles. Single tokens are cut, merged and
// joined as in paged_decode.cuh. What bounds it is the latency of a few dependent reads where caches are short, and else
// the reads of K, 16 bytes a lane from 32 rows at a time.
#pragma once

#include "paged_decode.cuh"

namespace cb200 {

constexpr int kF32Warps = 8, kF32Rows = 8;

struct F32Row { int token, head, pos, slot; };  // token -1: none

// kWords: 16-byte words of a head's row, rounded up to 4, 8, 16 or 32.
template <int kWords> __global__ void __launch_bounds__(32 * kF32Warps, 2) k_paged_fp32(PagedDecodeArgs p, int tokens_per_item) {
    constexpr int U = 32, R = kF32Rows, kAt = 32 / kWords, DP = kWords * 4 < 32 ? 32 : kWords * 4;
    __shared__ __align__(16) float q[R][kWords * 4];
    __shared__ __align__(16) float merge[kF32Warps][R][kWords * 4];
    __shared__ float2 warp_ml[kF32Warps][R];
    __shared__ F32Row rows[R];
    const PagedArgs& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, words = a.dim / 4;
    asm volatile("griddepcontrol.launch_dependents;" :::);

    float m[R], l[R], o[R][4];
    // Units [first, last) of `seen` for the rows of one slot (the others see nothing).
    const auto attend = [&](int slot, int kvh, const SeenUnits<U>& seen, int first, int last) {
        int pos[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
            pos[r] = rows[r].slot == slot ? rows[r].pos : -1;
#pragma unroll
            for (int c = 0; c < 4; ++c) o[r][c] = 0.f;
        }
        const int vrow = lane / kWords, vword = lane % kWords;
        for (int u = first + warp; u < last; u += kF32Warps) {
            const int j = seen.begin(u) + lane, entry = int(a.by_page.div(uint32_t(j))), row = j - entry * a.page;
            int id = j <= seen.pos && entry < a.width ? __ldg(a.table + slot * a.ts + entry) : -1;
            if (id >= a.pages) id = -1;
            unsigned vis = 0;
#pragma unroll
            for (int r = 0; r < R; ++r) vis |= unsigned(id >= 0 && sees(pos[r], j, a.window, a.first)) << r;
            const int64_t voff = id * a.vp + row * a.vr + kvh * a.vh;
            const float* k = static_cast<const float*>(a.k) + (vis ? id * a.kp + row * a.kr + kvh * a.kh : 0);
            float s[R] = {};
#pragma unroll 4
            for (int c = 0; c < words; ++c) {
                const float4 kw = vis ? __ldg(reinterpret_cast<const float4*>(k) + c) : make_float4(0, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float4 qw = *reinterpret_cast<const float4*>(&q[r][4 * c]);
                    s[r] = fmaf(qw.x, kw.x, fmaf(qw.y, kw.y, fmaf(qw.z, kw.z, fmaf(qw.w, kw.w, s[r]))));
                }
            }
            bool grow = false;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                s[r] = (vis >> r) & 1 ? s[r] * a.scale_log2 : -INFINITY;
                grow |= s[r] > m[r] + 8.f;
            }
            if (__any_sync(0xffffffffu, grow))
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float top = fmaxf(m[r], warp_max(s[r]));
                    const float corr = m[r] == -INFINITY ? (l[r] == 0.f ? 0.f : 1.f) : fast_exp2(m[r] - top);
                    m[r] = top;
                    l[r] *= corr;
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[r][c] *= corr;
                }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                s[r] = fast_exp2(s[r] - (m[r] == -INFINITY ? 0.f : m[r]));
                l[r] += s[r];
            }
            const unsigned any = __ballot_sync(0xffffffffu, vis != 0);
#pragma unroll 4
            for (int pass = 0; pass < kWords; ++pass) {
                const int e = pass * kAt + vrow;
                const int64_t off = __shfl_sync(0xffffffffu, voff, e);
                float4 v = make_float4(0, 0, 0, 0);
                if ((any >> e & 1) && vword < words) v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(a.v) + off) + vword);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float w = __shfl_sync(0xffffffffu, s[r], e);
                    if (w != 0.f) {  // a row that does not see the key takes nothing from it, whatever it holds
                        o[r][0] = fmaf(w, v.x, o[r][0]);
                        o[r][1] = fmaf(w, v.y, o[r][1]);
                        o[r][2] = fmaf(w, v.z, o[r][2]);
                        o[r][3] = fmaf(w, v.w, o[r][3]);
                    }
                }
            }
        }
    };
    // Merges the warps; finishes the rows of `slot`, or leaves the item's part.
    const auto end = [&](int slot, bool complete, int number) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            l[r] = warp_sum(l[r]);
#pragma unroll
            for (int c = 0; c < 4; ++c)
                for (int off = kWords; off < 32; off <<= 1) o[r][c] += __shfl_xor_sync(0xffffffffu, o[r][c], off);
        }
        if (lane < kWords)
#pragma unroll
            for (int r = 0; r < R; ++r) *reinterpret_cast<float4*>(&merge[warp][r][4 * lane]) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
        if (lane == 0)
#pragma unroll
            for (int r = 0; r < R; ++r) warp_ml[warp][r] = make_float2(m[r], l[r]);
        __syncthreads();
        for (int e = threadIdx.x; e < R * kWords * 4; e += 32 * kF32Warps) {
            const int r = e / (kWords * 4), d = e % (kWords * 4);
            const F32Row row = rows[r];
            if (d >= a.dim || row.token < 0 || row.slot != slot) continue;
            float top = -INFINITY, sum = 0.f, x = 0.f;
#pragma unroll
            for (int v = 0; v < kF32Warps; ++v) top = fmaxf(top, warp_ml[v][r].x);
#pragma unroll
            for (int v = 0; v < kF32Warps; ++v) {
                const float2 ml = warp_ml[v][r];
                const float weight = part_weight(ml.x, ml.y, top);
                sum += ml.y * weight;
                x += merge[v][r][d] * weight;
            }
            if (complete) {
                const HeadEnd he = head_end(top, sum, sink_log2<float>(a.sinks, a.sinks_fp32, row.head));
                static_cast<float*>(a.out)[row.token * a.ot + row.head * a.oh + d] = he.inv == 0.f ? 0.f : x * he.c * he.inv;
                if (a.lse && d == 0) a.lse[int64_t(row.token) * a.heads + row.head] = he.lse;
            } else {
                const int64_t at = int64_t(number) * R + r;
                p.parts[at * DP + d] = x;
                if (d == 0) p.part_ml[at] = make_float2(top, sum);
            }
        }
        __syncthreads();
    };
    const auto load_rows = [&](int token0, int tokens, int kvh, int block, int known_slot) {
        if (threadIdx.x < R) {
            F32Row row{-1, 0, -1, -1};
            const int per = min(a.group - block * R, R);  // heads of a token in this item
            const int t = threadIdx.x / per, h = threadIdx.x % per;
            if (t < tokens) {
                row.slot = known_slot >= 0 ? known_slot : slot_of(a.starts, a.slots, token0 + t);
                row.head = kvh * a.group + block * R + h;
                if (row.slot >= 0) {
                    row.token = token0 + t;
                    const int held = held_rows(a.lengths, row.slot, a.width, a.page);
                    row.pos = a.starts ? held - a.starts[row.slot + 1] + row.token : held - 1;
                }
            }
            rows[threadIdx.x] = row;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < R * a.dim; e += 32 * kF32Warps) {
            const int r = e / a.dim, d = e % a.dim;
            const F32Row row = rows[r];
            q[r][d] = row.token < 0 ? 0.f : static_cast<const float*>(a.q)[row.token * a.qt + row.head * a.qh + d];
        }
        __syncthreads();
    };

    if (a.starts) {  // a prompt: one CTA per item, the slots of its tokens one after another
        const int items = a.kv * p.blocks, item = blockIdx.x % items, kvh = item / p.blocks;
        const int token0 = int(blockIdx.x) / items * tokens_per_item, tokens = min(tokens_per_item, a.tokens - token0);
        load_rows(token0, tokens, kvh, item % p.blocks, -1);
        int slot = -1;
        for (int r = 0; r < R; ++r) {
            if (rows[r].token < 0 || rows[r].slot == slot) continue;
            slot = rows[r].slot;
            int first = INT_MAX, last = -1;
            for (int e = 0; e < R; ++e)
                if (rows[e].slot == slot) {
                    first = min(first, rows[e].pos);
                    last = max(last, rows[e].pos);
                }
            SeenUnits<U> seen;
            if (last >= 0) seen.set(a, max(first, 0), last);
            attend(slot, kvh, seen, 0, seen.units);
            end(slot, true, 0);
        }
        return;
    }
    const LinePart<U> part = cut_line<U, kF32Warps>(p);
    const int kvh = part.item / p.blocks;
    each_item<U>(p, part, [&](const LinePart<U>& at, int first, int last) {
        load_rows(at.slot, 1, kvh, part.item % p.blocks, at.slot);
        attend(at.slot, kvh, at.seen, at.u, at.u + last - first);
    }, [&](const LinePart<U>& at, bool complete, int number) { end(at.slot, complete, number); });
}

}  // namespace cb200
