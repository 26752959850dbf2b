// C entries of the operators over a paged key-value cache and of logits processing (include/chroma_b200.h): checks of
// their arguments, choice of kernel, launches. Nothing here allocates or synchronises.
#include "../../include/chroma_b200.h"

#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <cstdio>
#include <stdexcept>
#include <string>
#include <type_traits>
#include <utility>

#include "logits.cuh"
#include "paged.cuh"
#include "paged_decode.cuh"
#include "paged_fp32.cuh"
#include "paged_prompt.cuh"
#include "pages.cuh"

namespace {

using namespace cb200;

struct OpsValueError : std::runtime_error { using std::runtime_error::runtime_error; };

template <typename F> int guarded_op(char* err, size_t n, F&& f) {
    const char* text = "unknown native error";
    int code = CHROMA_B200_RUNTIME;
    std::string held;
    try {
        f();
        return CHROMA_B200_OK;
    } catch (const OpsValueError& e) {
        code = CHROMA_B200_VALUE;
        held = e.what();
        text = held.c_str();
    } catch (const std::exception& e) {
        held = e.what();
        text = held.c_str();
    } catch (...) {
    }
    if (err && n) std::snprintf(err, n, "%s", text);
    return code;
}

void want(bool ok, const char* what) {
    if (!ok) throw OpsValueError(what);
}

void check(cudaError_t status, const char* what) {
    if (status != cudaSuccess) throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(status));
}

template <typename... Params, typename... Args>
void launch_clusters(cudaStream_t s, int ctas, dim3 grid, dim3 block, size_t smem, void (*kernel)(Params...), Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(ctas);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctas > 1 ? 1 : 0;
    check(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...), "kernel launch");
}

template <typename... Params, typename... Args>
void launch(cudaStream_t s, dim3 grid, dim3 block, size_t smem, void (*kernel)(Params...), Args&&... args) {
    launch_clusters(s, 1, grid, block, smem, kernel, std::forward<Args>(args)...);
}

// A kernel that may start while the one before it drains; it waits for that one's results itself.
template <typename... Params, typename... Args>
void launch_after(cudaStream_t s, dim3 grid, dim3 block, void (*kernel)(Params...), Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    check(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...), "kernel launch");
}

constexpr int kDevices = 64;

int current_device() {
    int device = 0;
    check(cudaGetDevice(&device), "device");
    return device;
}

int sm_count() {
    static std::atomic<int> known[kDevices];
    const int device = current_device();
    int n = device < kDevices ? known[device].load(std::memory_order_relaxed) : 0;
    if (!n) {
        check(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device), "device attribute");
        if (device < kDevices) known[device].store(n, std::memory_order_relaxed);
    }
    return n;
}

// Lets a kernel have up to `bytes` of dynamic shared memory, the most that any call of it asks for: set once per device, so that no
// call takes away what another thread's has been given.
template <auto Kernel> void allow_smem(size_t bytes) {
    static std::atomic<bool> done[kDevices];
    const int device = current_device();
    if (device < kDevices && done[device].load(std::memory_order_acquire)) return;
    check(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)), "smem attribute");
    if (device < kDevices) done[device].store(true, std::memory_order_release);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

constexpr int kMaxRows = 1 << 30;  // positions of a slot: row numbers stay well inside 32 bits

size_t element(int storage) { return storage == CHROMA_B200_BF16 ? 2 : 4; }

void check_pages(const chroma_b200_pages* p) {
    want(p && p->keys && p->values && p->table && p->lengths, "null argument");
    want(p->storage == CHROMA_B200_FP32 || p->storage == CHROMA_B200_BF16, "pools are fp32 or bf16");
    want(p->layers > 0 && p->pages > 0 && p->page_rows > 0 && p->kv_heads > 0 && p->slots > 0 && p->width > 0,
         "empty pool or table");
    const int64_t size = int64_t(element(p->storage));
    want(p->head_dim > 0 && p->head_dim * size % 16 == 0 && p->head_dim <= 128,
         "head_dim: at most 128, and a multiple of 16 bytes");
    want(int64_t(p->width) * p->page_rows <= kMaxRows, "a table of more than 2^30 positions");
    want(int64_t(p->page_rows) * p->kv_heads * p->head_dim * size <= (int64_t(1) << 29), "a page of more than 512 MB");
    want(int64_t(p->pages) * p->layers < (int64_t(1) << 30), "more than 2^30 pages in all layers");
    want(aligned16(p->keys) && aligned16(p->values), "pools must be 16-byte aligned");
    for (int i = 0; i < 4; ++i)
        want(p->key_strides[i] * size % 16 == 0 && p->value_strides[i] * size % 16 == 0,
             "strides of the pools must be multiples of 16 bytes");
}

template <typename F> void by_type(int storage, F&& f) {
    if (storage == CHROMA_B200_BF16) f(__nv_bfloat16());
    else f(float());
}

PoolArgs pool_args(const chroma_b200_pages& p) {
    const int64_t per = 16 / int64_t(element(p.storage));
    PoolArgs a{};
    a.k = static_cast<uint4*>(p.keys);
    a.v = static_cast<uint4*>(p.values);
    a.kl = p.key_strides[0] / per, a.kp = p.key_strides[1] / per, a.kr = p.key_strides[2] / per, a.kh = p.key_strides[3] / per;
    a.vl = p.value_strides[0] / per, a.vp = p.value_strides[1] / per, a.vr = p.value_strides[2] / per, a.vh = p.value_strides[3] / per;
    a.layers = p.layers;
    a.heads = p.kv_heads;
    a.run = int(p.head_dim / per);
    if (a.kh == a.run && a.vh == a.run) a.run *= a.heads, a.heads = 1, a.kh = a.vh = a.run;  // a row is one run
    return a;
}

// Timeouts of bounded waits on this device, read by chroma_b200_operators_check.
__device__ unsigned g_error;

unsigned* error_word() {
    static std::atomic<void*> known[kDevices];
    const int device = current_device();
    void* at = device < kDevices ? known[device].load(std::memory_order_relaxed) : nullptr;
    if (!at) {
        check(cudaGetSymbolAddress(&at, g_error), "error word");
        if (device < kDevices) known[device].store(at, std::memory_order_relaxed);
    }
    return static_cast<unsigned*>(at);
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Tensor maps of bf16 boxes whose rows are 64 values, 128-byte swizzle; of a pool: one head, `rows` rows of one page. False
// where the strides are none that the TMA engine takes.
bool bf16_map(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    static const EncodeTiled encode = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q{};
        check(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q), "cuTensorMapEncodeTiled");
        if (!p || q != cudaDriverEntryPointSuccess) throw std::runtime_error("cuTensorMapEncodeTiled unavailable");
        return reinterpret_cast<EncodeTiled>(p);
    }();
    const cuuint32_t step[4] = {1, 1, 1, 1};
    for (int i = 0; i + 1 < rank; ++i)
        if (strides[i] == 0 || strides[i] >> 40 || strides[i] % 16) return false;
    return aligned16(base) && encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, cuuint32_t(rank), const_cast<void*>(base), dims, strides, box, step,
                                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool page_map(CUtensorMap* map, const void* pool, const PagedArgs& a, int64_t kp, int64_t kr, int64_t kh, int rows) {
    const cuuint64_t dims[4] = {cuuint64_t(a.dim), cuuint64_t(a.kv), cuuint64_t(a.page), cuuint64_t(a.pages)};
    const cuuint64_t strides[3] = {cuuint64_t(kh * 2), cuuint64_t(kr * 2), cuuint64_t(kp * 2)};
    const cuuint32_t box[4] = {64, 1, cuuint32_t(rows), 1};
    return bf16_map(map, pool, 4, dims, strides, box);
}

// How single tokens are laid out, and their workspace: partial results of two items per CTA, and each CTA's join.
struct DecodeSpace {
    int grid, tiles, pad, blocks, storage;  // CTAs at most, tiles of 8 heads in an item, padded head row, items per kv head
    int64_t parts, ml, bytes;
    DecodeSpace(int heads, int kv, int dim, int type) {
        const int group = heads / kv;
        storage = type;
        tiles = group > 8 && storage == CHROMA_B200_BF16 ? 2 : 1;
        pad = dim <= 32 ? 32 : dim <= 64 ? 64 : 128;
        blocks = (group + 8 * tiles - 1) / (8 * tiles);
        grid = sm_count() * 4;
        const int64_t rows = int64_t(2) * grid * 8 * tiles;
        parts = rows * pad * 4;
        ml = rows * 8;
        bytes = parts + ml + int64_t(grid) * 16;
    }
    // One CTA per item where its warps have one or two units anyway, where there are so many items that they even out,
    // and where the heads alone outnumber the CTAs; prompts have an item per rows in fp32, and no cuts. The host knows the
    // positions that the table could name, not those that are held. (One sequence of 160 positions, 8/1 heads of 16: 8.4 us;
    // cut and joined, as in a table for 131,072, 10.7.)
    bool whole(int slots, int kv, int64_t positions, const void* starts) const {
        return starts || positions <= 256 || int64_t(slots) * kv * blocks >= int64_t(8) * grid || int64_t(kv) * blocks > sm_count();
    }
    void place(PagedDecodeArgs& p, const chroma_b200_attention& g) const {
        want(g.workspace && g.workspace_bytes >= bytes, "workspace too small");
        p.parts = static_cast<float*>(g.workspace);
        p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(g.workspace) + parts);
        p.joins = reinterpret_cast<int4*>(static_cast<char*>(g.workspace) + parts + ml);
    }
};

template <int DC, int NT> void decode_join(const PagedDecodeArgs& p, int grid, cudaStream_t s) {
    if (p.whole) return;
    // A warp joins few parts by itself; where a line has few sequences for its CTAs, their items have many parts (a CTA
    // joins them: one sequence of 32,768 25 us, by a warp 33; 64 sequences of 64-256 27 us by warps, by CTAs 29).
    const int line = grid / (p.a.kv * p.blocks);
    if (p.a.slots >= line / 4) launch_after(s, dim3(unsigned(grid), NT), dim3(256), k_paged_join<__nv_bfloat16, 32 * DC, true>, p, 8 * NT);
    else launch_after(s, dim3(unsigned(grid), 8 * NT), dim3(256), k_paged_join<__nv_bfloat16, 32 * DC, false>, p, 8 * NT);
}

template <int DC, int NT> void decode_bf16(PagedDecodeArgs& p, int64_t items, cudaStream_t s) {
    const PagedArgs& a = p.a;
    CUtensorMap kmap, vmap;
    if constexpr (DC != 1) {
        using Ring = DecodeRing<DC>;
        p.box = a.page % Ring::U == 0 ? Ring::U : 16;
        if (p.full && a.page % 16 == 0 && page_map(&kmap, a.k, a, a.kp, a.kr, a.kh, p.box) && page_map(&vmap, a.v, a, a.vp, a.vr, a.vh, p.box)) {
            const int grid = p.whole ? int(items) : sm_count() * 2;
            p.least = 2 * Ring::kWarps;
            check(cudaFuncSetAttribute(k_paged_decode_tma<DC, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring::kSmem), "smem attribute");
            launch(s, dim3(unsigned(grid)), dim3(32 * Ring::kWarps), Ring::kSmem, k_paged_decode_tma<DC, NT>, p, kmap, vmap);
            return decode_join<DC, NT>(p, grid, s);
        }
    }
    using Regs = DecodeRegs<DC, NT>;
    const auto kernel = a.page % 16 == 0 ? k_paged_decode<DC, NT, true> : k_paged_decode<DC, NT, false>;
    const int grid = p.whole ? int(items) : sm_count() * Regs::kCtas;
    p.least = 2 * Regs::kWarps;
    launch(s, dim3(unsigned(grid)), dim3(32 * Regs::kWarps), 0, kernel, p);
    decode_join<DC, NT>(p, grid, s);
}

void decode(const PagedArgs& a, const chroma_b200_attention& g, int storage, cudaStream_t s) {
    const DecodeSpace space(a.heads, a.kv, a.dim, storage);
    PagedDecodeArgs p{};
    p.a = a;
    p.blocks = space.blocks;
    p.error = error_word();
    const int64_t lines = int64_t(a.kv) * p.blocks, items = a.slots * lines;
    want(items < kMaxRows, "more than 2^30 heads");
    p.whole = space.whole(a.slots, a.kv, int64_t(a.width) * a.page, a.starts);
    const int64_t size = int64_t(element(storage));
    p.full = a.dim == space.pad;
    p.kp = a.kp * size, p.kr = a.kr * size, p.vp = a.vp * size, p.vr = a.vr * size;
    p.q_vector = aligned16(a.q) && a.qt * size % 16 == 0 && a.qh * size % 16 == 0;
    if (!p.whole) space.place(p, g);
    const auto by_dim = [&](auto dc) {
        if (space.tiles == 2) decode_bf16<decltype(dc)::value, 2>(p, items, s);
        else decode_bf16<decltype(dc)::value, 1>(p, items, s);
    };
    if (space.pad == 32) by_dim(std::integral_constant<int, 1>());
    else if (space.pad == 64) by_dim(std::integral_constant<int, 2>());
    else by_dim(std::integral_constant<int, 4>());
}

void attention_fp32(const PagedArgs& a, const chroma_b200_attention& g, cudaStream_t s) {
    const DecodeSpace space(a.heads, a.kv, a.dim, CHROMA_B200_FP32);
    PagedDecodeArgs p{};
    p.a = a;
    p.blocks = space.blocks;
    p.least = kF32Warps;
    const int64_t lines = int64_t(a.kv) * p.blocks, items = a.slots * lines;
    const int per_item = a.starts && a.group < kF32Rows ? kF32Rows / a.group : 1;
    p.whole = space.whole(a.slots, a.kv, int64_t(a.width) * a.page, a.starts);
    int64_t blocks = a.starts ? (int64_t(a.tokens) + per_item - 1) / per_item * lines : p.whole ? items : sm_count() * 2;
    // Items of a prompt that leave SMs without work share them out, as long as every warp may have two units (16 tokens after
    // 8,000, 16/2 heads of 64: 47 us, without 174; after 4,000 with 64/8 heads 70 and 102). By the positions that the table could
    // name: three prompts of 5-61 after 37, 8/1 heads of 16, take 8.6 us, and 12.5 in a table for 131,072.
    p.share = 1;
    if (a.starts)
        while (p.share < 8 && 2 * p.share * blocks <= 2 * sm_count() && int64_t(a.width) * a.page >= 2 * p.share * 2 * kF32Warps * 32) p.share *= 2;
    blocks *= p.share;
    want(blocks < kMaxRows, "more than 2^30 heads");
    if (!p.whole) space.place(p, g);
    const auto run = [&](auto words) {
        constexpr int W = decltype(words)::value, DP = W * 4 < 32 ? 32 : W * 4;
        constexpr int smem = sizeof(F32Space<W>);
        if (smem > 48 * 1024) check(cudaFuncSetAttribute(k_paged_fp32<W>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "smem attribute");
        launch_clusters(s, p.share, dim3(unsigned(blocks)), dim3(32 * kF32Warps), smem, k_paged_fp32<W>, p, per_item);
        if (p.whole) return;
        if (a.slots >= blocks / lines / 4) launch_after(s, dim3(unsigned(blocks), 1), dim3(256), k_paged_join<float, DP, true>, p, kF32Rows);
        else launch_after(s, dim3(unsigned(blocks), kF32Rows), dim3(256), k_paged_join<float, DP, false>, p, kF32Rows);
    };
    if (a.dim <= 16) run(std::integral_constant<int, 4>());
    else if (a.dim <= 32) run(std::integral_constant<int, 8>());
    else if (a.dim <= 64) run(std::integral_constant<int, 16>());
    else run(std::integral_constant<int, 32>());
}

// How prompts are laid out, and their workspace: partial results of every split of every item.
struct PromptSpace {
    int64_t items, parts = 0, bytes = 0;  // items: at least as many as there are
    int tiles, splits = 1;                // tiles: pairs of tiles of rows, an item for each key-value head
    PromptSpace(int tokens, int group, int slots, int kv, int dim, int64_t positions) {
        tiles = int(int64_t(tokens) * group / 256) + std::max(1, std::min(slots, tokens));
        items = int64_t(tiles) * kv;
        // Fewer items than half the SMs share the SMs out, as long as four key tiles of the positions that the table could name are
        // left to each split. (Two prompts of 100, 64/8 heads of 64: 10.4 us; in a table for 131,072, with splits, 24.8.)
        const int64_t most = positions / (4 * kPrTile), share = sm_count() / items;
        if (share > 1 && most > 1) splits = int(share < most ? share : most);
        if (splits > 1) {
            parts = items * splits * 256 * (dim <= 64 ? 64 : 128) * 4;
            bytes = parts + items * splits * 256 * 8;
        }
    }
};

template <int H> void prompt_bf16(PagedPromptArgs& p, const chroma_b200_attention& g, cudaStream_t s) {
    const PagedArgs& a = p.a;
    CUtensorMap kmap{}, vmap{};
    p.box = 0;
    for (int rows = kPrTile; rows >= 8 && !p.box; rows /= 2)
        if (a.page % rows == 0) p.box = rows;
    if (p.box && !(page_map(&kmap, a.k, a, a.kp, a.kr, a.kh, p.box) && page_map(&vmap, a.v, a, a.vp, a.vr, a.vh, p.box))) p.box = 0;
    CUtensorMap qmap{};
    const cuuint64_t dims[3] = {cuuint64_t(a.dim), cuuint64_t(a.heads), cuuint64_t(a.tokens)};
    const cuuint64_t strides[2] = {cuuint64_t(a.qh * 2), cuuint64_t(a.qt * 2)};
    const cuuint32_t box[3] = {64, cuuint32_t(a.group), cuuint32_t(kPrTile / (a.group <= kPrTile ? a.group : kPrTile))};
    p.q_box = kPrTile % a.group == 0 && bf16_map(&qmap, a.q, 3, dims, strides, box);
    const PromptSpace space(a.tokens, a.group, a.slots, a.kv, a.dim, int64_t(a.width) * a.page);
    p.tiles = space.tiles;
    p.splits = space.splits;
    p.by_splits = FastDiv(uint32_t(p.splits));
    if (p.splits > 1) {
        want(g.workspace && g.workspace_bytes >= space.bytes, "workspace too small");
        p.parts = static_cast<float*>(g.workspace);
        p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(g.workspace) + space.parts);
    }
    const int64_t work = space.items * p.splits;
    const int grid = int(work < sm_count() ? work : sm_count());
    check(cudaFuncSetAttribute(k_paged_prompt<H>, cudaFuncAttributeMaxDynamicSharedMemorySize, PromptShape<H>::kSmem), "smem attribute");
    launch(s, dim3(unsigned(grid)), dim3(kPrThreads), PromptShape<H>::kSmem, k_paged_prompt<H>, p, qmap, kmap, vmap);
    if (p.splits > 1) launch_after(s, dim3(unsigned(space.items * 8)), dim3(256), k_prompt_join<H>, p);
}

void prompt(const PagedArgs& a, const chroma_b200_attention& g, int storage, cudaStream_t s) {
    PagedPromptArgs p{};
    p.a = a;
    p.by_group = FastDiv(uint32_t(a.group));
    p.by_kv = FastDiv(uint32_t(a.kv));
    p.error = error_word();
    const int64_t size = int64_t(element(storage));
    p.q_vector = aligned16(a.q) && a.qt * size % 16 == 0 && a.qh * size % 16 == 0;
    // A result may be written over its query: each row's is read before, once.
    const auto end = [&](const void* at, int64_t token, int64_t head) {
        return reinterpret_cast<uintptr_t>(at) + ((a.tokens - 1) * token + (a.heads - 1) * head + a.dim) * size;
    };
    p.over_q = reinterpret_cast<uintptr_t>(a.q) < end(a.out, a.ot, a.oh) && reinterpret_cast<uintptr_t>(a.out) < end(a.q, a.qt, a.qh);
    p.out_vector = aligned16(a.out) && a.ot * size % 16 == 0 && a.oh * size % 16 == 0;
    if (a.dim <= 64) prompt_bf16<1>(p, g, s);
    else prompt_bf16<2>(p, g, s);
}

// `list` and `count` as the launch before leaves them on the device.
void copy_pages(const chroma_b200_pages& p, const int* list, const int* count, cudaStream_t s) {
    const PoolArgs a = pool_args(p);
    const int64_t parts = (int64_t(p.page_rows) * a.heads * a.run + 1023) / 1024;
    const int64_t columns = (8 * sm_count() + parts - 1) / parts;
    launch_after(s, dim3(unsigned(columns), unsigned(parts)), dim3(256), k_pages_copy, a, list, count);
}

// One CTA decides about pages and slots that fit its shared memory, and a table that it reads in a few rounds. The decisions
// alone, steps and compaction, with pages of 1 KB: 4,096 pages and 128 slots 10.7 and 12.8 us, with several launches 11.3 and 16.9;
// 16,384 and 512: 25.1 and 39.4, 23.0 and 35.3; 32,768 and 1,000: 59.9 and 80.9, 57.4 and 70.1; 32,768 and 64: 44.0 and 33.3, 60.4 and
// 41.5. So it loses where pools and slots are both large, by 4 to 15%, and wins elsewhere by as much or more.
constexpr int kOneCtaPages = 32 * 1024, kOneCtaSlots = 1024;
bool one_cta(const chroma_b200_pages& p) {
    return p.pages <= kOneCtaPages && p.slots <= kOneCtaSlots && int64_t(p.slots) * p.width <= 64 * 1024;
}

size_t marks_bytes(int pages, int slots) { return size_t(pages) * 4 + size_t(slots) * sizeof(SlotStep) + size_t(pages) * 2; }
template <auto Kernel> size_t shared_marks(const chroma_b200_pages& p) {
    allow_smem<Kernel>(marks_bytes(kOneCtaPages, kOneCtaSlots));
    return marks_bytes(p.pages, p.slots);
}

// Bytes of the best of every segment of every row: of k_logits, or of k_logits_rest and k_logits_heard.
int64_t logits_best_bytes(int64_t rows, int64_t vocab) { return rows * ((vocab + kLogitsShort - 1) / kLogitsShort + 1) * 8; }

// CTAs that share a row in k_logits_heard: one a SM in all (two a SM, with half the threads each, took 33 us for 64 rows where this
// takes 31, and 22 for twelve where this takes 16), and as many as it takes for every entry that can come to have a slot,
// and every word of bits a place; no more than there are long segments.
int heard_ctas(const chroma_b200_logits& g) {
    const int64_t words = (int64_t(g.vocab) + 31) / 32, come = (g.history ? int64_t(g.width) : 0) + (g.bias_ids ? g.biases : 0);
    int64_t ctas = sm_count() / g.rows, need = (words + kHeardWords - 1) / kHeardWords;
    if (come > kHeardMost) need = std::max(need, (words * 32 + kHeardMost - 1) / kHeardMost);
    ctas = std::max(ctas, need);
    return int(std::max<int64_t>(1, std::min(ctas, std::max(need, (words + 127) / 128))));
}

dim3 table_grid(const chroma_b200_pages& p) { return dim3(unsigned((p.width + 255) / 256), unsigned(p.slots)); }

void step_pages(const chroma_b200_pages* p, const int32_t* parents, const int32_t* counts, int32_t* new_table, int32_t* new_lengths,
                int32_t* info, void* workspace, int64_t workspace_bytes, bool cut, cudaStream_t s) {
    check_pages(p);
    want(parents && counts && new_table && new_lengths && info && workspace, "null argument");
    want(workspace_bytes >= chroma_b200_pages_workspace(p->pages, p->slots), "workspace too small");
    want((int64_t(p->page_rows) + 1) * p->slots < (int64_t(1) << 32), "page_rows * slots must be below 2^32");
    want(p->slots <= 65535, "at most 65,535 slots");
    StepArgs a{};
    a.table = p->table, a.ts = p->table_stride, a.lengths = p->lengths, a.parents = parents, a.counts = counts;
    a.new_table = new_table, a.new_lengths = new_lengths, a.info = info;
    a.keeper = static_cast<unsigned*>(workspace);
    a.free_list = static_cast<int*>(workspace) + p->pages;
    a.copies = a.free_list + p->pages;
    a.slots = p->slots, a.width = p->width, a.pages = p->pages, a.page = p->page_rows;
    a.cut = cut;
    if (one_cta(*p)) launch(s, dim3(1), dim3(1024), shared_marks<k_pages_step>(*p), k_pages_step, a);
    else {
        check(cudaMemsetAsync(a.keeper, 0, size_t(p->pages) * 4, s), "memset");
        launch(s, table_grid(*p), dim3(256), 0, k_pages_gather, a);
        launch(s, dim3(1), dim3(1024), 0, k_pages_assign, a);
    }
    copy_pages(*p, a.copies, a.copies + 3 * p->slots, s);
}

}  // namespace

extern "C" {

int chroma_b200_operators_check(void* stream, char* err, size_t err_len) {
    return guarded_op(err, err_len, [&] {
        unsigned word = 0;
        unsigned* at = error_word();
        const auto s = cudaStream_t(stream);
        check(cudaMemcpyAsync(&word, at, sizeof word, cudaMemcpyDeviceToHost, s), "error word");
        check(cudaStreamSynchronize(s), "operators");
        if (!word) return;
        check(cudaMemsetAsync(at, 0, sizeof word, s), "error word");
        throw std::runtime_error("a bounded wait inside an operator's kernel timed out; its outputs are incomplete");
    });
}

int chroma_b200_paged_append(const chroma_b200_pages* p, const void* new_keys, const void* new_values,
                             const int64_t* new_strides, const int32_t* starts, int32_t tokens, void* stream, char* err,
                             size_t err_len) {
    return guarded_op(err, err_len, [&] {
        check_pages(p);
        want(tokens >= 0 && new_strides, "null argument");
        want(starts || tokens == p->slots, "without starts there is one row per slot");
        if (!tokens) return;
        want(new_keys && new_values, "null argument");
        AppendArgs a{};
        a.nk = new_keys, a.nv = new_values;
        a.nkt = new_strides[0], a.nkh = new_strides[1], a.nvt = new_strides[2], a.nvh = new_strides[3];
        a.k = p->keys, a.v = p->values;
        a.kp = p->key_strides[1], a.kr = p->key_strides[2], a.kh = p->key_strides[3];
        a.vp = p->value_strides[1], a.vr = p->value_strides[2], a.vh = p->value_strides[3];
        a.table = p->table, a.ts = p->table_stride, a.lengths = p->lengths, a.starts = starts;
        a.slots = p->slots, a.width = p->width, a.pages = p->pages, a.page = p->page_rows, a.kv = p->kv_heads;
        a.dim = p->head_dim, a.tokens = tokens, a.by_page = FastDiv(uint32_t(p->page_rows));
        const int64_t size = int64_t(element(p->storage));
        a.by_run = FastDiv(uint32_t(p->head_dim * size / 16));
        int vector = aligned16(new_keys) && aligned16(new_values);
        for (int i = 0; i < 4; ++i) vector = vector && new_strides[i] * size % 16 == 0;
        by_type(p->storage, [&](auto t) {
            launch(cudaStream_t(stream), dim3(unsigned((tokens + kAppendWarps - 1) / kAppendWarps)), dim3(32 * kAppendWarps), 0, k_paged_append<decltype(t)>, a, vector);
        });
    });
}

int64_t chroma_b200_attention_workspace(const chroma_b200_pages* p, const chroma_b200_attention* g) {
    if (!p || !g || g->heads <= 0 || p->kv_heads <= 0 || g->heads % p->kv_heads || p->head_dim <= 0) return -1;
    try {
        if (g->starts && p->storage == CHROMA_B200_BF16)
            return PromptSpace(g->tokens, g->heads / p->kv_heads, p->slots, p->kv_heads, p->head_dim, int64_t(p->width) * p->page_rows).bytes;
        const DecodeSpace space(g->heads, p->kv_heads, p->head_dim, p->storage);
        return space.whole(p->slots, p->kv_heads, int64_t(p->width) * p->page_rows, g->starts) ? 0 : space.bytes;
    } catch (...) {
        return -1;
    }
}

int chroma_b200_paged_attention(const chroma_b200_pages* p, const chroma_b200_attention* g, void* stream, char* err,
                                size_t err_len) {
    return guarded_op(err, err_len, [&] {
        check_pages(p);
        want(g && g->tokens >= 0, "null argument");
        want(g->heads > 0 && g->heads % p->kv_heads == 0, "heads must be a multiple of kv_heads");
        want(g->starts || g->tokens == p->slots, "without starts there is one token per slot");
        want(g->first >= 0, "first must be nonnegative");
        want(g->scale > 0, "scale must be positive");
        want(int64_t(g->tokens) * g->heads <= kMaxRows, "more than 2^30 rows of queries");
        if (!g->tokens) return;
        want(g->q && g->out, "null argument");
        PagedArgs a{};
        a.k = p->keys, a.v = p->values;
        a.kp = p->key_strides[1], a.kr = p->key_strides[2], a.kh = p->key_strides[3];
        a.vp = p->value_strides[1], a.vr = p->value_strides[2], a.vh = p->value_strides[3];
        a.table = p->table, a.ts = p->table_stride, a.lengths = p->lengths, a.starts = g->starts;
        a.slots = p->slots, a.width = p->width, a.pages = p->pages, a.page = p->page_rows, a.kv = p->kv_heads;
        a.dim = p->head_dim, a.by_page = FastDiv(uint32_t(p->page_rows));
        a.q = g->q, a.out = g->out, a.lse = g->lse, a.sinks = g->sinks, a.sinks_fp32 = g->sinks_fp32;
        a.qt = g->q_strides[0], a.qh = g->q_strides[1], a.ot = g->out_strides[0], a.oh = g->out_strides[1];
        a.tokens = g->tokens, a.heads = g->heads, a.group = g->heads / p->kv_heads;
        a.window = g->window, a.first = g->first, a.scale_log2 = g->scale * kLog2e;
        const auto s = cudaStream_t(stream);
        if (p->storage == CHROMA_B200_FP32) attention_fp32(a, *g, s);
        else if (g->starts) prompt(a, *g, p->storage, s);
        else decode(a, *g, p->storage, s);
    });
}

int64_t chroma_b200_pages_workspace(int32_t pages, int32_t slots) {
    return pages < 0 || slots < 0 ? -1 : (5 * int64_t(pages) + 3 * int64_t(slots) + 4) * 4;
}

int chroma_b200_step_pages(const chroma_b200_pages* p, const int32_t* parents, const int32_t* counts, int32_t* new_table,
                           int32_t* new_lengths, int32_t* info, void* workspace, int64_t workspace_bytes, void* stream,
                           char* err, size_t err_len) {
    return guarded_op(err, err_len, [&] { step_pages(p, parents, counts, new_table, new_lengths, info, workspace, workspace_bytes, true, cudaStream_t(stream)); });
}

int chroma_b200_step_pages_uncut(const chroma_b200_pages* p, const int32_t* parents, const int32_t* counts, int32_t* new_table,
                                 int32_t* new_lengths, int32_t* info, void* workspace, int64_t workspace_bytes, void* stream,
                                 char* err, size_t err_len) {
    return guarded_op(err, err_len, [&] { step_pages(p, parents, counts, new_table, new_lengths, info, workspace, workspace_bytes, false, cudaStream_t(stream)); });
}

int chroma_b200_compact_pages(const chroma_b200_pages* p, int32_t* new_table, int32_t* info, void* workspace,
                              int64_t workspace_bytes, void* stream, char* err, size_t err_len) {
    return guarded_op(err, err_len, [&] {
        check_pages(p);
        want(new_table && info && workspace, "null argument");
        want(workspace_bytes >= chroma_b200_pages_workspace(p->pages, p->slots), "workspace too small");
        want(p->slots <= 65535, "at most 65,535 slots");
        const auto s = cudaStream_t(stream);
        CompactArgs a{};
        a.table = p->table, a.ts = p->table_stride, a.lengths = p->lengths;
        a.new_table = new_table, a.info = info;
        a.held = static_cast<unsigned*>(workspace);
        a.copies = static_cast<int*>(workspace) + p->pages;
        a.holes = a.copies + 3 * p->pages + 1;
        a.slots = p->slots, a.width = p->width, a.pages = p->pages, a.page = p->page_rows;
        if (one_cta(*p)) launch(s, dim3(1), dim3(1024), shared_marks<k_compact>(*p), k_compact, a);
        else {
            check(cudaMemsetAsync(a.held, 0, size_t(p->pages) * 4, s), "memset");
            launch(s, table_grid(*p), dim3(256), 0, k_compact_mark, a);
            launch(s, dim3(1), dim3(1024), 0, k_compact_plan, a);
            launch(s, table_grid(*p), dim3(256), 0, k_compact_table, a);
        }
        copy_pages(*p, a.copies, a.copies + 3 * p->pages, s);
    });
}

int64_t chroma_b200_logits_workspace(int32_t rows, int32_t vocab) {
    return rows < 0 || vocab < 0 ? -1 : logits_best_bytes(rows, vocab) + int64_t(rows) * ((int64_t(vocab) + 31) / 32) * 4;
}

int chroma_b200_process_logits(const chroma_b200_logits* g, void* stream, char* err, size_t err_len) {
    return guarded_op(err, err_len, [&] {
        want(g && g->rows >= 0 && g->vocab > 0 && g->vocab <= kMaxRows, "null argument or empty vocabulary");
        want(g->storage == CHROMA_B200_FP32 || g->storage == CHROMA_B200_BF16, "logits are fp32 or bf16");
        want(!g->history || (g->lengths && g->width >= 0), "a history needs its lengths");
        want(!g->bias_ids || (g->bias && g->biases >= 0), "bias_ids need their bias");
        want(g->rows <= 65535, "at most 65,535 rows");
        if (!g->rows) return;
        want(g->logits && g->out, "null argument");
        want(!(g->argmax || g->history || g->bias_ids) || (g->workspace && g->workspace_bytes >= chroma_b200_logits_workspace(g->rows, g->vocab)),
             "workspace too small");
        const auto s = cudaStream_t(stream);
        LogitsArgs a{};
        a.logits = g->logits, a.out = g->out, a.history = g->history, a.lengths = g->lengths, a.prompts = g->prompts;
        a.repetition = g->repetition, a.presence = g->presence, a.frequency = g->frequency, a.temperature = g->temperature;
        a.bias_ids = g->bias_ids, a.bias = g->bias, a.mask = reinterpret_cast<const unsigned*>(g->mask);
        a.best = g->argmax ? static_cast<unsigned long long*>(g->workspace) : nullptr;
        a.stride = g->stride, a.out_stride = g->out_stride, a.history_stride = g->history_stride;
        a.bias_ids_stride = g->bias_ids_stride, a.bias_stride = g->bias_stride, a.mask_stride = g->mask_stride;
        a.vocab = g->vocab, a.width = g->width, a.biases = g->biases;
        const int64_t size = int64_t(element(g->storage));
        a.vector = aligned16(g->logits) && aligned16(g->out) && (g->rows == 1 || (g->stride * size % 16 == 0 && g->out_stride * size % 16 == 0));
        a.history_vector = aligned16(g->history) && (g->rows == 1 || g->history_stride % 4 == 0);
        // Long segments once they alone give every SM two CTAs (both measured beside kLogitsShort).
        const bool few = int64_t(g->rows) * ((g->vocab + kLogitsLong - 1) / kLogitsLong) < 2 * sm_count();
        const int short_segments = (g->vocab + kLogitsShort - 1) / kLogitsShort, long_segments = (g->vocab + kLogitsLong - 1) / kLogitsLong;
        by_type(g->storage, [&](auto t) {
            using T = decltype(t);
            const dim3 threads(kLogitsThreads), rest(unsigned(long_segments), unsigned(g->rows));
            if (few) {
                a.segments = short_segments;
                launch(s, dim3(unsigned(short_segments), unsigned(g->rows)), threads, 0, k_logits<T>, a);
                return;
            }
            a.segments = long_segments;
            if (!a.history && !a.bias_ids) return launch(s, rest, threads, 0, k_logits_rest<T>, a);
            a.special_stride = (g->vocab + 31) / 32;
            a.special = reinterpret_cast<unsigned*>(static_cast<char*>(g->workspace) + logits_best_bytes(g->rows, g->vocab));
            const int ctas = heard_ctas(*g);
            a.by_ctas = FastDiv(uint32_t(ctas));
            a.best_at = long_segments;
            a.segments += ctas;
            const int smem = int(sizeof(HeardTable)) + (a.special_stride + ctas - 1) / ctas * 4;
            allow_smem<k_logits_heard<T>>(sizeof(HeardTable) + kHeardWords * 4);
            launch(s, dim3(unsigned(ctas), unsigned(g->rows)), dim3(kHeardThreads), smem, k_logits_heard<T>, a);
            launch_after(s, rest, threads, k_logits_rest<T>, a);
        });
        if (g->argmax) launch_after(s, dim3(unsigned(g->rows)), dim3(32), k_logits_pick, a.best, a.segments, g->argmax);
    });
}

}  // extern "C"
