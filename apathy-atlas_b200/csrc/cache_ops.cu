// The operators around the paged K/V cache: attention that reads it, and its pages between two steps.  Argument checks, choice of
// kernel and launches; like the rest of the library it allocates nothing, does not synchronise and reads no device memory on the host.
#include "atlas_b200.h"

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>

#include "common.cuh"
#include "host_launch.hpp"
#include "kernel_attn.cuh"
#include "kernel_attn_mma.cuh"
#include "kernel_attn_tc.cuh"
#include "kernel_cache_pages.cuh"

namespace atlas {

int cache_device_status(uint32_t* out_word, int clear) {
    cudaError_t e = cudaMemcpyFromSymbol(out_word, g_status_word, sizeof(uint32_t));
    if (e == cudaSuccess && clear) {
        const uint32_t zero = 0;
        e = cudaMemcpyToSymbol(g_status_word, &zero, sizeof(uint32_t));
    }
    return cuda_status(e);
}

namespace {

constexpr int kMaxDevices = 64;
std::mutex g_attr_mutex;

// Dynamic shared memory above 48 KB is a setting of a kernel on a device: made at its first launch there.
template <typename K> int allow_smem(K kernel, int bytes, std::atomic<bool> (&done)[kMaxDevices]) {
    int dev = -1;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_status(e);
    if (dev < 0 || dev >= kMaxDevices) return ATLAS_B200_ERR_LIMIT;
    if (done[dev].load(std::memory_order_acquire)) return ATLAS_B200_OK;
    std::lock_guard<std::mutex> lock(g_attr_mutex);
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) done[dev].store(true, std::memory_order_release);
    return cuda_status(e);
}

template <typename... P, typename... A>
int launch_dependent(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, uint32_t cluster, A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
}

// ---------------------------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------------------------
thread_local uint32_t t_attn_shape[4] = {0, 0, 0, 0};

// room for a cut of every range: more than any GPU this library runs on has SMs, twice
constexpr size_t ATTN_CUT_BYTES = 1024 * sizeof(AttnCut);
constexpr uint32_t ATTN_MAX_CTAS = 1024;

uint32_t attn_dim(uint32_t head_dim) { return head_dim <= 64 ? 64u : head_dim <= 128 ? 128u : 256u; }

int check_attention(const atlas_b200_attention_desc& d) {
    if (d.q_heads == 0 || d.kv_heads == 0 || d.q_heads % d.kv_heads || d.head_dim == 0 || d.head_dim % 32 || d.head_dim > 256 || d.block_size == 0 ||
        d.table_stride == 0 || d.n_pages == 0)
        return ATLAS_B200_ERR_DIMS;
    if (d.cache_dtype != ATLAS_B200_CACHE_BF16 && d.cache_dtype != ATLAS_B200_CACHE_E4M3) return ATLAS_B200_ERR_DIMS;
    if (uint64_t(d.q_heads) * d.head_dim > d.q_row_stride || uint64_t(d.q_heads) * d.head_dim > d.out_row_stride) return ATLAS_B200_ERR_DIMS;
    if (!(d.softmax_scale > 0.0f) || !std::isfinite(d.softmax_scale) || !(d.k_scale > 0.0f) || !std::isfinite(d.k_scale) || !(d.v_scale > 0.0f) ||
        !std::isfinite(d.v_scale) || !std::isfinite(d.softmax_scale * d.k_scale * ATTN_LOG2E))
        return ATLAS_B200_ERR_DIMS;
    if (d.cache_dtype == ATLAS_B200_CACHE_BF16 && (d.k_scale != 1.0f || d.v_scale != 1.0f)) return ATLAS_B200_ERR_DIMS;
    // rows of the cache and places of a sequence are counted in 31 bits
    if (uint64_t(d.n_pages) * d.block_size >= (1ull << 31) || uint64_t(d.table_stride) * d.block_size >= (1ull << 31) || d.n_seqs >= (1u << 24) ||
        d.n_tokens >= (1u << 31) || uint64_t(d.n_tokens) * (d.q_heads / d.kv_heads) >= (1ull << 31))
        return ATLAS_B200_ERR_LIMIT;
    if (!d.q || !d.out || !d.k_cache || !d.v_cache || !d.block_table || !d.cu_q || !d.kv_len) return ATLAS_B200_ERR_NULL;
    if (!aligned(d.q, 4) || d.q_row_stride % 2 || !aligned(d.out, 2) || !aligned(d.k_cache, 16) || !aligned(d.v_cache, 16) || !aligned(d.block_table, 4) ||
        !aligned(d.cu_q, 4) || !aligned(d.kv_len, 4) || !aligned(d.lse, 4) || !aligned(d.ws, 32))
        return ATLAS_B200_ERR_ALIGN;
    return ATLAS_B200_OK;
}

AttnParams attention_params(const atlas_b200_attention_desc& d) {
    AttnParams p{};
    p.q = static_cast<const uint16_t*>(d.q);
    p.out = static_cast<uint16_t*>(d.out);
    p.lse = d.lse;
    p.k_cache = static_cast<const uint8_t*>(d.k_cache);
    p.v_cache = static_cast<const uint8_t*>(d.v_cache);
    p.block_table = d.block_table; p.cu_q = d.cu_q; p.kv_len = d.kv_len;
    p.cuts = static_cast<AttnCut*>(d.ws);
    p.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(d.ws) + ATTN_CUT_BYTES);
    p.n_seqs = d.n_seqs; p.n_tokens = d.n_tokens; p.n_pages = d.n_pages; p.table_stride = d.table_stride;
    p.q_heads = d.q_heads; p.kv_heads = d.kv_heads; p.head_dim = d.head_dim; p.block_size = d.block_size; p.group = d.q_heads / d.kv_heads;
    p.page_div = attn_divisor(d.block_size);
    p.group_div = attn_divisor(p.group);
    p.q_row_stride = d.q_row_stride; p.out_row_stride = d.out_row_stride;
    p.scale = d.softmax_scale; p.k_scale = d.k_scale; p.v_scale = d.v_scale;
    return p;
}

// What an item costs besides its tiles, in tiles of its kernel.  256 sequences of up to 1000 tokens, mma.sync: 0 / 1 / 2 / 3 of them give
// 112 / 101 / 96.5 / 97.3 us; tcgen05, 8192 tokens by themselves: 1 / 2 / 3 give 569 / 475 / 476 us (head_dim 256: 860 / 877 / 893).
constexpr uint32_t MMA_EXTRA = 2;
constexpr uint32_t tc_extra(uint32_t dim) { return dim <= 128 ? 2u : 1u; }

constexpr uint32_t log2_of(uint32_t n) { return n <= 1 ? 0u : 1u + log2_of(n / 2); }
AttnShape shape_of(const AttnParams& p, uint32_t rows, uint32_t keys, uint32_t extra) {
    return attn_shape(p.group, log2_of(rows), log2_of(keys), extra, uint64_t(p.table_stride) * p.block_size, uint64_t(p.n_tokens) * p.group);
}

// Whole items, where the CTA that has the most of them takes less than what equal ranges take with the scratch that cuts need and its
// join: some twelve tiles' time.  The sequences' lengths, which the host does not know, are taken for three quarters of the longest one's
// on the average: whole items wait for the longest.  (One or two items a CTA: beyond, equal ranges lose little.)
bool whole_items_pay(uint64_t items, uint64_t places, uint64_t ctas) {
    const uint64_t rounds = (items + ctas - 1) / ctas;
    return rounds <= 2 && rounds * places <= items * places * 3 / (4 * ctas) + 12;
}

// Scratch for the cuts and the pieces of up to `ctas` ranges.
size_t cuts_bytes(uint32_t ctas, uint32_t block_rows, uint32_t dim) { return ATTN_CUT_BYTES + size_t(ctas) * 2 * attn_part_floats(block_rows, dim) * sizeof(float); }

// Rows that a KV head has in the longest chunk.
uint64_t chunk_rows(const atlas_b200_attention_desc& d) { return uint64_t(std::min(d.max_q_len, d.n_tokens)) * (d.q_heads / d.kv_heads); }

// The mma.sync form: how many CTAs, and whether each takes whole items.  (Nothing is cut up to MMA_WHOLE_TILES tiles.)
constexpr uint64_t MMA_WHOLE_TILES = 4;
struct MmaPlan {
    uint32_t ctas, by_item, least, tile, block_rows, cluster_log2;
    size_t ws_bytes, most_ws_bytes;      // that it takes; that fewer sequences or shorter ones may take
};
MmaPlan plan_mma(const atlas_b200_attention_desc& d, uint32_t sms, bool scratch) {
    const uint32_t dim = attn_dim(d.head_dim);
    const uint64_t rows = chunk_rows(d);
    MmaPlan r{};
    r.block_rows = rows <= 8 ? 8u : 16u;
    const bool fp8 = d.cache_dtype == ATLAS_B200_CACHE_E4M3;
    const uint32_t row_bytes = dim * (fp8 ? 1u : 2u), resident = std::min(sms, ATTN_MAX_CTAS / 3) * uint32_t(attn::attn_mma_ctas(int(row_bytes), fp8, r.block_rows == 8u ? 1 : 2));
    const uint64_t items = uint64_t(d.n_seqs) * d.kv_heads * std::max<uint64_t>((rows + r.block_rows - 1) / r.block_rows, 1);
    r.tile = uint32_t(attn::MMA_WARPS) * (row_bytes <= 128u ? 32u : 16u);
    const uint64_t tiles = std::max<uint64_t>((uint64_t(d.max_kv_len) + r.tile - 1) / r.tile, 1);
    // Few items: a cluster each, of as many CTAs as there are tiles for (four a CTA, where SMs take more than one) and places on the SMs; unless
    // that leaves a CTA more than eight tiles, which the line's equal ranges share better, given scratch.
    const auto wider = [&] { return items << (r.cluster_log2 + 1); };
    while (r.cluster_log2 < 3 && wider() <= resident && (wider() <= sms ? 2ull : 8ull) << r.cluster_log2 <= tiles) ++r.cluster_log2;
    if (scratch && tiles > 8ull << r.cluster_log2) r.cluster_log2 = 0;
    // 64 sequences of 500 tokens, 8 KV heads of 128, 29.8 us whole and 35.0 cut; 64 of 300, 22.0 and 26.5; 40 of 700, 33.4 and 31.3; over E4M3
    // 40 of 700, 22.9 and 29.1.
    r.by_item = !scratch || r.cluster_log2 || tiles <= MMA_WHOLE_TILES || whole_items_pay(items, tiles + MMA_EXTRA, resident);      // (no scratch: nothing is cut)
    r.least = r.by_item ? 1u : 4u;
    const uint64_t places = r.by_item ? items : (items * (tiles + MMA_EXTRA) + r.least - 1) / r.least;
    r.ctas = uint32_t(std::min<uint64_t>(r.cluster_log2 ? items : resident, std::max<uint64_t>(places, 1)));
    r.most_ws_bytes = tiles <= MMA_WHOLE_TILES ? 0 : cuts_bytes(resident, r.block_rows, dim);
    r.ws_bytes = r.by_item ? 0 : r.most_ws_bytes;
    return r;
}

template <int DP, bool FP8, int RT> int launch_mma_rows(AttnParams p, const MmaPlan& plan, cudaStream_t st) {
    using C = attn::MmaCfg<DP, FP8, RT>;
    static std::atomic<bool> done[kMaxDevices] = {};
    const int rc = allow_smem(attn::attn_mma_kernel<DP, FP8, RT>, C::SMEM, done);
    if (rc) return rc;
    p.ctas = plan.ctas; p.least_tiles = plan.least; p.by_item = plan.by_item; p.cluster_log2 = plan.cluster_log2;
    p.shape = shape_of(p, C::ROWS, C::TILE, MMA_EXTRA);
    const int rc2 = launch_dependent(attn::attn_mma_kernel<DP, FP8, RT>, plan.ctas << plan.cluster_log2, attn::MMA_THREADS, C::SMEM, st, 1u << plan.cluster_log2, p);
    if (rc2 || plan.by_item || plan.ctas < 2) return rc2;
    return launch_dependent(attn_join_kernel<C::ROWS, DP, FP8>, dim3(plan.ctas - 1, ATTN_JOIN_Y), ATTN_JOIN_THREADS, 0, st, 1u, p);
}

template <int DP, bool FP8> int launch_mma(const AttnParams& p, const MmaPlan& plan, cudaStream_t st) {
    return plan.block_rows == 8 ? launch_mma_rows<DP, FP8, 1>(p, plan, st) : launch_mma_rows<DP, FP8, 2>(p, plan, st);
}

// The tcgen05 form.  It reads pages in boxes of the largest power of two that divides page and tile, or row by row where that is less than a
// swizzle atom's eight rows; and Q and the outputs in sixteen bytes.
constexpr uint64_t TC_WHOLE_TILES = 2;
struct TcPlan {
    uint32_t ctas, by_item, least, box_rows;
    size_t ws_bytes, most_ws_bytes;      // as above
};
uint32_t tc_box_rows(uint32_t block_size) {
    uint32_t r = attn::TC_KEYS;
    while (block_size % r) r /= 2;
    return r;
}
bool rows_pay_for_tc(const atlas_b200_attention_desc& d) {
    // Rows of a KV head from which on the tensor cores' 256-row blocks pay, although most of such a block is empty.  Sequences of 4000 tokens, 8 KV
    // heads of 128, this form / mma.sync.  BF16, 12 rows: 4 sequences 28 / 21 us, 16 54 / 56, 64 188 / 180; 20 rows, two blocks to
    // mma.sync: 16 sequences 54 / 95 (the latter over pages of 5).  E4M3, whose tiles are converted by four warps, 12 rows: 31 / 23, 70 / 53, 249 / 147; 20 rows: 32 / 36, 71 / 84, 252 / 270;
    // 32 rows: 34 / 36, 71 / 86, 255 / 273: from 17 rows on this form would be the shorter there too, by a seventh at most.
    // Over pages that are copied row by row it costs half as much again (pages of 5, 16 sequences: BF16 head_dim 128, 20 rows 138 / 95, 48 rows
    // 141 / 136; head_dim 256, 20 rows 212 / 266; E4M3 head_dim 128, 20 rows 104 / 86, 48 rows 104 / 112; head_dim 256, 20 rows 190 / 169).
    const bool fp8 = d.cache_dtype == ATLAS_B200_CACHE_E4M3, boxes = tc_box_rows(d.block_size) >= 8;
    const uint64_t from = boxes ? (fp8 ? 32 : 16) : !fp8 && d.head_dim > 128 ? 16 : 48;
    return chunk_rows(d) > from;
}
bool takes_tc(const atlas_b200_attention_desc& d) {
    return rows_pay_for_tc(d) && aligned(d.q, 16) && aligned(d.out, 16) && d.q_row_stride % 8 == 0 && d.out_row_stride % 8 == 0;
}
TcPlan plan_tc(const atlas_b200_attention_desc& d, uint32_t sms) {
    sms = std::min(sms, ATTN_MAX_CTAS);
    const uint32_t dim = attn_dim(d.head_dim), block_rows = dim <= 128 ? 256u : 128u;
    const uint64_t items = uint64_t(d.n_seqs) * d.kv_heads * ((chunk_rows(d) + block_rows - 1) / block_rows);
    const uint64_t tiles = std::max<uint64_t>((uint64_t(d.max_kv_len) + attn::TC_KEYS - 1) / attn::TC_KEYS, 1);
    TcPlan r{};
    r.box_rows = tc_box_rows(d.block_size);
    // Two chunks of 512 over 1024 tokens, 8 KV heads of 128, 24.2 us whole and 42.3 cut; 300 over 300, 12.2 and 22.2; eight of 64 over
    // 2000, head_dim 64, 32.6 and 30.5.
    const uint64_t item = tiles + tc_extra(dim);
    r.by_item = tiles <= TC_WHOLE_TILES || whole_items_pay(items, item, sms);
    r.least = r.by_item ? 1u : 2u;
    const uint64_t places = r.by_item ? items : (items * item + r.least - 1) / r.least;
    r.ctas = uint32_t(std::min<uint64_t>(sms, std::max<uint64_t>(places, 1)));
    r.most_ws_bytes = tiles <= TC_WHOLE_TILES ? 0 : cuts_bytes(sms, block_rows, dim);
    r.ws_bytes = r.by_item ? 0 : r.most_ws_bytes;
    return r;
}

template <int DP, bool FP8> int launch_tc(AttnParams p, const TcPlan& plan, cudaStream_t st) {
    using C = attn::TcCfg<DP, FP8>;
    static std::atomic<bool> done[kMaxDevices] = {};
    const int rc = allow_smem(attn::attn_tc_kernel<DP, FP8>, C::SMEM, done);
    if (rc) return rc;
    CUtensorMap map_k, map_v;
    const uint64_t size = FP8 ? 1 : 2;
    const uint64_t dims[3] = {p.head_dim, p.kv_heads, uint64_t(p.n_pages) * p.block_size};
    const uint64_t strides[2] = {p.head_dim * size, uint64_t(p.kv_heads) * p.head_dim * size};
    const uint32_t box_rows = std::min(plan.box_rows, uint32_t(C::KEYS));
    const uint32_t box[3] = {FP8 ? uint32_t(DP) : 64u, 1u, std::max(box_rows, 8u)};   // (below eight: not used)
    const CUtensorMapDataType dt = FP8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const CUtensorMapSwizzle swz = FP8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B;
    if (!encode_tensor_map(&map_k, dt, 3, p.k_cache, dims, strides, box, swz) || !encode_tensor_map(&map_v, dt, 3, p.v_cache, dims, strides, box, swz))
        return ATLAS_B200_ERR_DIMS;
    p.ctas = plan.ctas; p.least_tiles = plan.least; p.by_item = plan.by_item; p.shape = shape_of(p, C::ROWS, attn::TC_KEYS, tc_extra(DP));
    const int rc2 = launch_dependent(attn::attn_tc_kernel<DP, FP8>, plan.ctas, C::THREADS, C::SMEM, st, 1u, map_k, map_v, p, box_rows);
    if (rc2 || plan.by_item || plan.ctas < 2) return rc2;
    return launch_dependent(attn_join_kernel<C::ROWS, DP, FP8>, dim3(plan.ctas - 1, ATTN_JOIN_Y), ATTN_JOIN_THREADS, 0, st, 1u, p);
}

// What is asked for does not shrink as sequences are added or grow, although fewer of them may be cut: a buffer for a server's largest batch
// does for all smaller ones.  (Which kernel runs also goes by the alignment of pointers that may not be set yet: enough for either where the
// rows alone would have it tcgen05.)
size_t attention_ws_bytes(const atlas_b200_attention_desc& d, uint32_t sms) {
    return std::max(plan_mma(d, sms, true).most_ws_bytes, rows_pay_for_tc(d) ? plan_tc(d, sms).most_ws_bytes : size_t(0));
}

int attention(const atlas_b200_attention_desc& d, cudaStream_t st) {
    if (d.n_seqs == 0 || d.n_tokens == 0) return ATLAS_B200_OK;
    const int bad = check_attention(d);
    if (bad) return bad;
    if (!device_is_sm100()) return ATLAS_B200_ERR_ARCH;
    const uint32_t sms = uint32_t(device_sm_count()), dim = attn_dim(d.head_dim);
    if (!d.ws && d.ws_bytes) return ATLAS_B200_ERR_WORKSPACE;
    if (takes_tc(d)) {
        TcPlan plan = plan_tc(d, sms);
        if (d.ws && d.ws_bytes < plan.ws_bytes) return ATLAS_B200_ERR_WORKSPACE;
        if (!d.ws && !plan.by_item) { plan.by_item = 1; plan.least = 1; }
        const bool fp8 = d.cache_dtype == ATLAS_B200_CACHE_E4M3;
        const AttnParams p = attention_params(d);
        t_attn_shape[0] = dim <= 128 ? 256 : 128; t_attn_shape[1] = plan.ctas; t_attn_shape[2] = plan.by_item; t_attn_shape[3] = attn::TC_KEYS;
        if (dim == 64) return fp8 ? launch_tc<64, true>(p, plan, st) : launch_tc<64, false>(p, plan, st);
        if (dim == 128) return fp8 ? launch_tc<128, true>(p, plan, st) : launch_tc<128, false>(p, plan, st);
        return fp8 ? launch_tc<256, true>(p, plan, st) : launch_tc<256, false>(p, plan, st);
    }
    const MmaPlan plan = plan_mma(d, sms, d.ws != nullptr);
    if (d.ws && d.ws_bytes < plan.ws_bytes) return ATLAS_B200_ERR_WORKSPACE;
    const bool fp8 = d.cache_dtype == ATLAS_B200_CACHE_E4M3;
    const AttnParams p = attention_params(d);
    t_attn_shape[0] = plan.block_rows; t_attn_shape[1] = plan.ctas << plan.cluster_log2; t_attn_shape[2] = plan.by_item; t_attn_shape[3] = plan.tile;
    if (dim == 64) return fp8 ? launch_mma<64, true>(p, plan, st) : launch_mma<64, false>(p, plan, st);
    if (dim == 128) return fp8 ? launch_mma<128, true>(p, plan, st) : launch_mma<128, false>(p, plan, st);
    return fp8 ? launch_mma<256, true>(p, plan, st) : launch_mma<256, false>(p, plan, st);
}

// ---------------------------------------------------------------------------------------------
// pages
// ---------------------------------------------------------------------------------------------
size_t round256(size_t n) { return (n + 255) / 256 * 256; }

size_t pages_ws_bytes(const atlas_b200_cache_desc& d, uint32_t n) {
    return round256(size_t(d.n_seqs) * 4) + round256(size_t(n) * 24) + round256(size_t(d.n_pages) * 4) + 256;
}

int check_pages(const atlas_b200_cache_desc& d, uint32_t n, bool copies, pages::PagesParams& p) {
    if (d.n_pages == 0 || d.block_size == 0 || d.table_stride == 0 || d.n_seqs == 0) return ATLAS_B200_ERR_DIMS;
    if (copies && (d.page_bytes == 0 || d.page_bytes % d.block_size || d.page_bytes % 16)) return ATLAS_B200_ERR_DIMS;
    if (d.n_pages >= (1u << 31) || d.n_seqs >= (1u << 31) || uint64_t(d.table_stride) * d.block_size >= (1ull << 31) || n >= (1u << 24) || d.n_bases > 65535u)
        return ATLAS_B200_ERR_LIMIT;
    if (!d.refcount || !d.block_table || !d.seq_len || !d.ws || (copies && d.n_bases && !d.bases)) return ATLAS_B200_ERR_NULL;
    if (!aligned(d.refcount, 4) || !aligned(d.block_table, 4) || !aligned(d.seq_len, 4) || !aligned(d.bases, 8) || !aligned(d.ws, 16)) return ATLAS_B200_ERR_ALIGN;
    if (d.ws_bytes < pages_ws_bytes(d, n)) return ATLAS_B200_ERR_WORKSPACE;
    p.bases = d.bases;
    p.refcount = d.refcount; p.block_table = d.block_table; p.seq_len = d.seq_len;
    p.n_bases = d.n_bases; p.n_pages = d.n_pages; p.block_size = d.block_size; p.table_stride = d.table_stride; p.n_seqs = d.n_seqs;
    p.page_bytes = d.page_bytes;
    uint8_t* ws = static_cast<uint8_t*>(d.ws);
    p.claim = reinterpret_cast<int32_t*>(ws);
    p.entry = reinterpret_cast<int32_t*>(ws + round256(size_t(d.n_seqs) * 4));
    p.list = reinterpret_cast<int32_t*>(ws + round256(size_t(d.n_seqs) * 4) + round256(size_t(n) * 24));
    p.count = reinterpret_cast<int32_t*>(ws + round256(size_t(d.n_seqs) * 4) + round256(size_t(n) * 24) + round256(size_t(d.n_pages) * 4));
    return ATLAS_B200_OK;
}

}  // namespace
}  // namespace atlas

using namespace atlas;

extern "C" {

int atlas_b200_paged_attention(const atlas_b200_attention_desc* desc, void* stream) {
    if (!desc) return ATLAS_B200_ERR_NULL;
    return attention(*desc, static_cast<cudaStream_t>(stream));
}

size_t atlas_b200_paged_attention_ws_bytes(const atlas_b200_attention_desc* desc) {
    if (!desc || desc->kv_heads == 0 || desc->q_heads % desc->kv_heads || desc->n_seqs == 0 || desc->n_tokens == 0) return 0;
    return attention_ws_bytes(*desc, uint32_t(device_sm_count()));
}

int atlas_b200_last_attention_shape(uint32_t out[4]) {
    if (!out) return ATLAS_B200_ERR_NULL;
    for (int i = 0; i < 4; ++i) out[i] = t_attn_shape[i];
    return ATLAS_B200_OK;
}

size_t atlas_b200_cache_ws_bytes(const atlas_b200_cache_desc* desc, uint32_t n) { return desc ? pages_ws_bytes(*desc, n) : 0; }

int atlas_b200_cache_append(const atlas_b200_cache_desc* desc, const int32_t* seqs, const int32_t* n_new, uint32_t n, uint32_t max_tokens,
                            long long* slot_mapping, int32_t* status, void* stream) {
    if (!desc) return ATLAS_B200_ERR_NULL;
    if (n == 0 && max_tokens == 0) return ATLAS_B200_OK;
    if ((n && (!seqs || !n_new)) || (max_tokens && !slot_mapping)) return ATLAS_B200_ERR_NULL;
    if (max_tokens >= (1u << 31)) return ATLAS_B200_ERR_LIMIT;
    if (!aligned(seqs, 4) || !aligned(n_new, 4) || !aligned(slot_mapping, 8) || !aligned(status, 4)) return ATLAS_B200_ERR_ALIGN;
    pages::PagesParams p{};
    const int bad = check_pages(*desc, n, false, p);
    if (bad) return bad;
    return launch_dependent(pages::append_kernel, 1, pages::PLAN_THREADS, 0, static_cast<cudaStream_t>(stream), 1u, p, seqs, n_new, n, max_tokens, slot_mapping, status);
}

int atlas_b200_cache_fork(const atlas_b200_cache_desc* desc, const int32_t* src, const int32_t* dst, uint32_t n, int32_t* status, void* stream) {
    if (!desc) return ATLAS_B200_ERR_NULL;
    if (n == 0) return ATLAS_B200_OK;
    if (!src || !dst) return ATLAS_B200_ERR_NULL;
    if (!aligned(src, 4) || !aligned(dst, 4) || !aligned(status, 4)) return ATLAS_B200_ERR_ALIGN;
    pages::PagesParams p{};
    const int bad = check_pages(*desc, n, true, p);
    if (bad) return bad;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int rc = launch_dependent(pages::fork_plan_kernel, 1, pages::PLAN_THREADS, 0, st, 1u, p, src, dst, n, status);
    if (rc) return rc;
    return launch_dependent(pages::fork_copy_kernel, dim3(n, std::max(desc->n_bases, 1u)), pages::COPY_THREADS, 0, st, 1u, p, src, dst);
}

int atlas_b200_cache_free(const atlas_b200_cache_desc* desc, const int32_t* seqs, uint32_t n, void* stream) {
    if (!desc) return ATLAS_B200_ERR_NULL;
    if (n == 0) return ATLAS_B200_OK;
    if (!seqs) return ATLAS_B200_ERR_NULL;
    if (!aligned(seqs, 4)) return ATLAS_B200_ERR_ALIGN;
    pages::PagesParams p{};
    const int bad = check_pages(*desc, n, false, p);
    if (bad) return bad;
    return launch_dependent(pages::free_kernel, n, pages::FREE_THREADS, 0, static_cast<cudaStream_t>(stream), 1u, p, seqs);
}

int atlas_b200_cache_compact(const atlas_b200_cache_desc* desc, int32_t* refcount_out, int32_t* block_table_out, int32_t* page_map, int32_t* n_used, void* stream) {
    if (!desc || !refcount_out || !block_table_out || !page_map || !n_used) return ATLAS_B200_ERR_NULL;
    if (!aligned(refcount_out, 4) || !aligned(block_table_out, 4) || !aligned(page_map, 4) || !aligned(n_used, 4)) return ATLAS_B200_ERR_ALIGN;
    pages::PagesParams p{};
    const int bad = check_pages(*desc, 0, true, p);
    if (bad) return bad;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int rc = launch_dependent(pages::compact_plan_kernel, 1, pages::PLAN_THREADS, 0, st, 1u, p, refcount_out, page_map, n_used);
    if (rc) return rc;
    return launch_dependent(pages::compact_move_kernel, uint32_t(device_sm_count()) * 4, pages::COPY_THREADS, 0, st, 1u, p, page_map, block_table_out);
}

}  // extern "C"
