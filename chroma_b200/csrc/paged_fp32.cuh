// fp32 attention over a paged cache, single tokens and prompts, on the FMA pipe (tensor-core products of fp32 operands would
// keep 11 or 8 of their 24 bits).
//
// An item is up to 8 rows that share a key-value head: query heads of one token, or, where a key-value head has fewer than
// 8 of them, of several consecutive tokens. Units of 32 positions are dealt to the 8 warps of a CTA, and each warp works on
// its own. The unit's keys are copied to shared memory, 64 values of a row at a time, row by row; then a lane has one key: it
// walks the key's row there and multiplies each 16-byte word with the same words of the 8 query rows, which all lanes read
// from the same place, so a score needs no exchange between lanes. (Rows of 64 bytes are read by their lanes directly.)
// Values are read with a row spread over `kWords` lanes, the 8 weights of a key in two words of shared memory. Single tokens
// are cut, merged and joined as in paged_decode.cuh. Few items of a prompt after a long cache are each shared by the CTAs of a
// cluster, which merge through one another's shared memory.
//
// What bounds it: where caches are short, the latency of five dependent reads; else the latency of a unit's copies, which
// nothing hides but the other warps. A warp waits for its keys as soon as it has asked for them, and reads the values after the
// weights. 64 sequences of 500-2,000 positions with 64/8 heads of 64 take 109 us, 12 TFLOP/s, where their bytes take 51, the
// load pipe's work (about 400 cycles of an SM for 32 keys and 64 values) 28 and the FMA's issue 18; with each lane reading its
// own key from global memory, and weights passed by shuffles, they took 143. Two of 30,000-60,000 with 8/2 heads of 128: 78 us
// (bytes 28); two prompts of 1,000 with 16/4 heads of 64: 301 us; 16 tokens after 8,000, 16/2 heads of 64: 47 us. One sequence of
// 160 with 8 heads of 16: 8.2 us one call after another. At 128 registers, which let two CTAs share an SM, every width spills
// (132 bytes stored, 88 loaded a thread).
#pragma once

#include <limits.h>

#include "paged_decode.cuh"

namespace cb200 {

constexpr int kF32Warps = 8, kF32Rows = 8;

struct F32Row { int token, head, pos, slot; };  // token -1: none

// A warp's part of shared memory; the merge of the warps reuses the keys' place.
template <int kWords> struct F32Warp {
    static constexpr int kChunk = kWords < 16 ? kWords : 16;  // 16-byte words of a row at a time
    static constexpr int kStride = 4 * kChunk + 4;            // floats between keys: lanes that read a word each meet all banks
    union {
        float keys[32 * kStride];
        float merge[kF32Rows][4 * kWords];
    };
    float weights[32][kF32Rows];
    int64_t places[32][2];  // elements from the pools' start to the rows of the unit's keys and values
};
template <int kWords> struct F32Space {
    F32Warp<kWords> warps[kF32Warps];
    float q[kF32Rows][4 * kWords];
    float2 warp_ml[kF32Warps][kF32Rows];
    F32Row rows[kF32Rows];
};

// The float at the same place of shared memory in a CTA of the cluster.
__device__ __forceinline__ float mate_value(const float* p, int rank) {
    float x;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(cluster_addr(p, uint32_t(rank))) : "memory");
    return x;
}

// kWords: 16-byte words of a head's row, rounded up to 4, 8, 16 or 32.
template <int kWords> __global__ void __launch_bounds__(32 * kF32Warps, 2) k_paged_fp32(const __grid_constant__ PagedDecodeArgs p, int tokens_per_item) {
    constexpr int U = 32, R = kF32Rows, kAt = 32 / kWords, DP = kWords * 4 < 32 ? 32 : kWords * 4;
    constexpr int kChunk = F32Warp<kWords>::kChunk, kStride = F32Warp<kWords>::kStride, kKeysAt = 32 / kChunk;
    extern __shared__ __align__(16) uint8_t f32_smem[];
    F32Space<kWords>& sm = *reinterpret_cast<F32Space<kWords>*>(f32_smem);
    const PagedArgs& a = p.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, words = a.dim / 4;
    F32Warp<kWords>& mine = sm.warps[warp];
    asm volatile("griddepcontrol.launch_dependents;" :::);

    // ---- what this CTA has: tokens of a prompt, or a part of the line of single tokens
    const bool prompt = a.starts;
    const int share = p.share, mate = share > 1 ? blockIdx.x % share : 0, mates_block = share > 1 ? blockIdx.x / share : blockIdx.x;
    const int items = a.kv * p.blocks, item = mates_block % items, kvh = item / p.blocks, block = item % p.blocks;
    LinePart<U> part{};
    int token0 = 0;
    if (prompt) token0 = mates_block / items * tokens_per_item;
    else part = cut_line<U, kF32Warps>(p);
    LinePart<U> at = part;
    int4 join = make_int4(0, 0, 0, 0);
    int done = 0, slot = -1, next_row = 0;
    bool loaded = false;
    while (true) {
        // ---- the next piece: rows of one slot, and units of what they see
        if (!prompt && done >= part.count) break;
        if (!prompt || !loaded) {
            __syncthreads();
            if (threadIdx.x < R) {
                F32Row row{-1, 0, -1, -1};
                const int per = min(a.group - block * R, R);  // heads of a token in this item
                const int t = threadIdx.x / per, token = (prompt ? token0 : at.slot) + t;
                if (prompt ? t < tokens_per_item && token < a.tokens : t == 0) {
                    row.slot = prompt ? slot_of(a.starts, a.slots, token) : at.slot;
                    row.head = kvh * a.group + block * R + threadIdx.x % per;
                    if (row.slot >= 0) {
                        row.token = token;
                        row.pos = length_of(a.lengths, row.slot) - (prompt ? a.starts[row.slot + 1] - token : 1);
                    }
                }
                sm.rows[threadIdx.x] = row;
            }
            __syncthreads();
            for (int e = threadIdx.x; e < R * 4 * kWords; e += 32 * kF32Warps) {
                const int r = e / (4 * kWords), d = e % (4 * kWords);
                const F32Row row = sm.rows[r];
                sm.q[r][d] = row.token < 0 || d >= a.dim ? 0.f : static_cast<const float*>(a.q)[row.token * a.qt + row.head * a.qh + d];
            }
            __syncthreads();
            loaded = true;
        }
        SeenUnits<U> seen;
        int first = 0, last = 0, number = 0, lowest = INT_MAX;  // position of the piece's rows; seen.pos is the highest
        unsigned of_slot = 0;                                   // its rows
        for (int e = 0; e < R; ++e) of_slot |= unsigned(sm.rows[e].token >= 0) << e;
        bool complete = true;
        if (prompt) {
            while (next_row < R && (sm.rows[next_row].token < 0 || sm.rows[next_row].slot == slot)) ++next_row;
            if (next_row == R) break;
            slot = sm.rows[next_row].slot;
            int high = -1;
            for (int e = 0; e < R; ++e)
                if (sm.rows[e].token >= 0 && sm.rows[e].slot == slot) {
                    lowest = min(lowest, sm.rows[e].pos);
                    high = max(high, sm.rows[e].pos);
                } else of_slot &= ~(1u << e);
            if (high >= 0) seen.set(a, max(lowest, 0), high);
            last = seen.units;
        } else {
            slot = at.slot;
            seen = at.seen;
            lowest = seen.pos;
            const int take = min(part.count - done, seen.units - at.u);
            first = at.u;
            last = first + take;
            complete = first == 0 && take == seen.units;
            number = 2 * blockIdx.x + (done > 0 ? 1 : 0);
            if (!complete && first == 0) {
                const int64_t end = part.begin + done + seen.units;  // one past the item's last unit
                join = make_int4(slot, item, int((end * part.ctas - 1) / part.total) - int(blockIdx.x) / items, number);
            }
            done += take;
            at.u += take;
            if (at.u >= seen.units) at.next_slot(a);
        }

        // ---- its units, 8 warps of each CTA in turn
        float m[R], l[R], o[R][4];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) o[r][c] = 0.f;
        }
        for (int u = first + mate * kF32Warps + warp; u < last; u += share * kF32Warps) {
            const int j = seen.begin(u) + lane, entry = int(a.by_page.div(uint32_t(j))), row = j - entry * a.page;
            int id = j <= seen.pos && entry < a.width ? __ldg(a.table + slot * a.ts + entry) : -1;
            if (id >= a.pages) id = -1;
            const int j0 = j - lane;
            unsigned vis = id >= 0 ? of_slot : 0u;  // as it is where every row sees the whole unit
            if (j0 + U - 1 > lowest || (a.window > 0 && seen.pos - j0 >= a.window && j0 + U > a.first))
                for (int r = 0; r < R; ++r)
                    if (!sees(sm.rows[r].pos, j, a.window, a.first)) vis &= ~(1u << r);
            const unsigned any = __ballot_sync(0xffffffffu, vis != 0);
            mine.places[lane][0] = vis ? id * a.kp + row * a.kr + kvh * a.kh : 0;
            mine.places[lane][1] = vis ? id * a.vp + row * a.vr + kvh * a.vh : 0;
            __syncwarp();
            float s[R] = {};
            const auto score = [&](int c, const float4& kw) {  // word c of the row
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float4 qw = *reinterpret_cast<const float4*>(&sm.q[r][4 * c]);
                    s[r] = fmaf(qw.x, kw.x, fmaf(qw.y, kw.y, fmaf(qw.z, kw.z, fmaf(qw.w, kw.w, s[r]))));
                }
            };
            if constexpr (kWords == 4) {
                const float4* k = reinterpret_cast<const float4*>(static_cast<const float*>(a.k) + mine.places[lane][0]);
                float4 kw[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) kw[c] = vis && c < words ? __ldg(k + c) : make_float4(0, 0, 0, 0);
#pragma unroll
                for (int c = 0; c < 4; ++c) score(c, kw[c]);
            } else
#pragma unroll 1
            for (int chunk = 0; chunk < kWords; chunk += kChunk) {
#pragma unroll 4
                for (int pass = 0; pass < kChunk; ++pass) {
                    const int e = pass * kKeysAt + lane / kChunk, c = lane % kChunk;
                    const bool ok = (any >> e & 1) && chunk + c < words;
                    const float* from = static_cast<const float*>(a.k) + mine.places[e][0] + (ok ? 4 * (chunk + c) : 0);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(mine.keys + e * kStride + 4 * c)), "l"(from), "r"(ok ? 16 : 0) : "memory");
                }
                cp_async_commit();
                cp_async_wait<0>();
                __syncwarp();
#pragma unroll 4
                for (int c = 0; c < kChunk; ++c) score(chunk + c, *reinterpret_cast<const float4*>(mine.keys + lane * kStride + 4 * c));
                __syncwarp();
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
            *reinterpret_cast<float4*>(mine.weights[lane]) = make_float4(s[0], s[1], s[2], s[3]);
            *reinterpret_cast<float4*>(mine.weights[lane] + 4) = make_float4(s[4], s[5], s[6], s[7]);
            __syncwarp();
            const int vword = lane % kWords;
#pragma unroll 4
            for (int pass = 0; pass < kWords; ++pass) {
                const int e = pass * kAt + lane / kWords;
                float4 v = make_float4(0, 0, 0, 0);
                if ((any >> e & 1) && vword < words) v = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(a.v) + mine.places[e][1]) + vword);
                const float4 w0 = *reinterpret_cast<const float4*>(mine.weights[e]), w1 = *reinterpret_cast<const float4*>(mine.weights[e] + 4);
                const float w[R] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (w[r] != 0.f) {  // a row that does not see the key takes nothing from it, whatever it holds
                        o[r][0] = fmaf(w[r], v.x, o[r][0]);
                        o[r][1] = fmaf(w[r], v.y, o[r][1]);
                        o[r][2] = fmaf(w[r], v.z, o[r][2]);
                        o[r][3] = fmaf(w[r], v.w, o[r][3]);
                    }
            }
            __syncwarp();
        }

        // ---- the warps are merged; rows of the slot are finished, or the item's part is left
#pragma unroll
        for (int r = 0; r < R; ++r) {
            l[r] = warp_sum(l[r]);
#pragma unroll
            for (int c = 0; c < 4; ++c)
                for (int off = kWords; off < 32; off <<= 1) o[r][c] += __shfl_xor_sync(0xffffffffu, o[r][c], off);
        }
        if (lane < kWords)
#pragma unroll
            for (int r = 0; r < R; ++r) *reinterpret_cast<float4*>(&mine.merge[r][4 * lane]) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
        if (lane == 0)
#pragma unroll
            for (int r = 0; r < R; ++r) sm.warp_ml[warp][r] = make_float2(m[r], l[r]);
        __syncthreads();
        if (share > 1) cluster_sync_all();
        for (int e = threadIdx.x + mate * 32 * kF32Warps; e < R * kWords * 4; e += share * 32 * kF32Warps) {
            const int r = e / (kWords * 4), d = e % (kWords * 4);
            const F32Row row = sm.rows[r];
            if (d >= a.dim || row.token < 0 || row.slot != slot) continue;
            float top = -INFINITY, sum = 0.f, x = 0.f;
            if (share > 1) {  // the warps of all CTAs, in their order
                for (int c = 0; c < share; ++c)
#pragma unroll
                    for (int v = 0; v < kF32Warps; ++v) top = fmaxf(top, mate_value(&sm.warp_ml[v][r].x, c));
                for (int c = 0; c < share; ++c)
#pragma unroll
                    for (int v = 0; v < kF32Warps; ++v) {
                        const float total = mate_value(&sm.warp_ml[v][r].y, c), weight = part_weight(mate_value(&sm.warp_ml[v][r].x, c), total, top);
                        sum += total * weight;
                        x += mate_value(&sm.warps[v].merge[r][d], c) * weight;
                    }
            } else {
#pragma unroll
                for (int v = 0; v < kF32Warps; ++v) top = fmaxf(top, sm.warp_ml[v][r].x);
#pragma unroll
                for (int v = 0; v < kF32Warps; ++v) {
                    const float2 ml = sm.warp_ml[v][r];
                    const float weight = part_weight(ml.x, ml.y, top);
                    sum += ml.y * weight;
                    x += sm.warps[v].merge[r][d] * weight;
                }
            }
            if (complete) {
                const HeadEnd he = head_end(top, sum, sink_log2<float>(a.sinks, a.sinks_fp32, row.head));
                static_cast<float*>(a.out)[row.token * a.ot + row.head * a.oh + d] = he.inv == 0.f ? 0.f : x * he.c * he.inv;
                if (a.lse && d == 0) a.lse[int64_t(row.token) * a.heads + row.head] = he.lse;
            } else {
                const int64_t place = int64_t(number) * R + r;
                p.parts[place * DP + d] = x;
                if (d == 0) p.part_ml[place] = make_float2(top, sum);
            }
        }
        __syncthreads();
        if (share > 1) cluster_sync_all();
    }
    if (!prompt && !p.whole && threadIdx.x == 0) p.joins[blockIdx.x] = join;
}

}  // namespace cb200
