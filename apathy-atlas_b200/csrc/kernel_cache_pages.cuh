// Pages of the paged K/V cache between two steps: taken for new tokens, shared by forks, given back, moved together.
//
// All state is on the device, so that a captured step can take and give back pages: refcount [n_pages] (0: free), block_table
// [n_seqs, table_stride], seq_len [n_seqs]; a sequence of n tokens holds the first ceil(n / block_size) entries of its row.  A page that
// is part filled belongs to one sequence alone (a fork copies it), so that appending never writes where another sequence reads.
//
// What is taken is always the lowest free page, in the order of the call's entries: the same state and call give the same tables,
// whatever the timing.  That needs a prefix sum over the entries and one over the pages, which one CTA makes: 1024 threads look at 4096
// pages a turn and stop where they have found enough.  The copies (all layers' K and V, a list of base addresses on the device) are a
// second kernel over all SMs.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "common.cuh"

namespace atlas {
namespace pages {

constexpr int PLAN_THREADS = 1024, COPY_THREADS = 256;

struct PagesParams {
    const uint64_t* bases;        // [n_bases] device addresses of [n_pages][page_bytes]
    int32_t* refcount;
    int32_t* block_table;
    int32_t* seq_len;
    uint32_t n_bases, n_pages, block_size, table_stride, n_seqs;
    uint64_t page_bytes;
    // scratch
    int32_t* claim;               // [n_seqs] lowest entry of the call that names the sequence
    int32_t* entry;               // [n][6]
    int32_t* list;                // [n_pages] free pages found; or holes from the front and moved pages from the back
    int32_t* count;               // [4]
};

// Exclusive prefix sum over the CTA's threads of two counts in one word; `sum`: of all threads.
__device__ __forceinline__ uint64_t block_scan(uint64_t mine, uint64_t* sh, uint64_t& sum) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    uint64_t upto = mine;
#pragma unroll
    for (uint32_t o = 1; o < 32; o <<= 1) {
        const uint64_t v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += v;
    }
    __syncthreads();                                                         // the words of the scan before have been read
    if (lane == 31u) sh[warp] = upto;
    __syncthreads();
    if (warp == 0) {
        uint64_t w = sh[lane];
#pragma unroll
        for (uint32_t o = 1; o < 32; o <<= 1) {
            const uint64_t v = __shfl_up_sync(0xFFFFFFFFu, w, o);
            if (lane >= o) w += v;
        }
        sh[lane] = w;
    }
    __syncthreads();
    sum = sh[31];
    return upto - mine + (warp ? sh[warp - 1] : 0);
}

// The lowest free pages, up to `want` of them, into p.list in order; returns how many there are of those.
__device__ __forceinline__ uint32_t find_free(const PagesParams& p, uint64_t want, uint64_t* sh) {
    uint64_t found = 0;
    for (uint32_t base = 0; base < p.n_pages && found < want; base += 4 * PLAN_THREADS) {
        const uint32_t at = base + 4 * threadIdx.x;
        uint32_t is_free = 0;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            if (at + k < p.n_pages && p.refcount[at + k] == 0) is_free |= 1u << k;
        uint64_t sum;
        uint64_t to = found + block_scan(__popc(is_free), sh, sum);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            if ((is_free >> k) & 1u) {
                if (to < want) p.list[to] = int32_t(at + k);
                ++to;
            }
        found += sum;
    }
    __syncthreads();
    return uint32_t(found < want ? found : want);
}

// Which entry of the call speaks for a sequence: the lowest that names it.
__device__ __forceinline__ void claim_seqs(const PagesParams& p, const int32_t* seqs, uint32_t n) {
    for (uint32_t i = threadIdx.x; i < n; i += PLAN_THREADS)
        if (uint32_t(seqs[i]) < p.n_seqs) p.claim[seqs[i]] = 0x7FFFFFFF;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += PLAN_THREADS)
        if (uint32_t(seqs[i]) < p.n_seqs) atomicMin(p.claim + seqs[i], int32_t(i));
    __syncthreads();
}
__device__ __forceinline__ uint32_t pages_of(const PagesParams& p, uint64_t tokens) { return uint32_t((tokens + p.block_size - 1) / p.block_size); }

// ---- append ------------------------------------------------------------------------------------------------------
// Entry i gives sequence seqs[i] room for n_new[i] more tokens; slots of all entries' tokens in a row into slot_mapping.
// (Entries of the usual call are kept in shared memory: the second pass, a warp an entry, is a chain of the loads it makes.)
constexpr uint32_t APPEND_FIELDS = 6, APPEND_IN_SMEM = PLAN_THREADS;
__global__ void __launch_bounds__(PLAN_THREADS) append_kernel(PagesParams p, const int32_t* seqs, const int32_t* n_new, uint32_t n, uint32_t max_tokens,
                                                              long long* slot_mapping, int32_t* status) {
    __shared__ uint64_t sh[32];
    __shared__ int32_t entry_s[APPEND_FIELDS * APPEND_IN_SMEM];
    int32_t* const entry = n <= APPEND_IN_SMEM ? entry_s : p.entry;
    pdl_release();
    pdl_wait();
    seqs = pdl_after(seqs); n_new = pdl_after(n_new); p.refcount = pdl_after(p.refcount); p.block_table = pdl_after(p.block_table); p.seq_len = pdl_after(p.seq_len);
    claim_seqs(p, seqs, n);
    const uint64_t room = uint64_t(p.table_stride) * p.block_size;
    uint64_t need_all = 0, tokens_all = 0;
    for (uint32_t base = 0; base < n; base += PLAN_THREADS) {
        const uint32_t i = base + threadIdx.x;
        int32_t say = ATLAS_B200_ERR_DIMS;
        uint32_t need = 0, add = 0, s = 0;
        uint64_t len = 0;
        if (i < n) {
            s = uint32_t(seqs[i]);
            add = n_new[i] > 0 ? uint32_t(n_new[i]) : 0u;
            if (s < p.n_seqs && __ldcg(p.claim + s) == int32_t(i) && n_new[i] >= 0 && p.seq_len[s] >= 0 && uint64_t(p.seq_len[s]) <= room) {
                len = uint32_t(p.seq_len[s]);
                if (len + add > room) say = ATLAS_B200_ERR_LIMIT;
                else { say = 0; need = pages_of(p, len + add) - pages_of(p, len); }
            }
        }
        // (tokens are counted in 64 bits of their own: a call may name more than 2^31)
        uint64_t sum, tok_sum;
        const uint64_t tok = tokens_all + block_scan(add, sh, tok_sum);
        if (say == 0 && tok + add > max_tokens) { say = ATLAS_B200_ERR_LIMIT; need = 0; }
        const uint64_t before = need_all + block_scan(need, sh, sum);
        if (i < n) {
            int32_t* const e = entry + APPEND_FIELDS * i;
            e[0] = say;
            e[1] = int32_t(before > 0x7FFFFFFFull ? 0x7FFFFFFFull : before);
            e[2] = int32_t(need);
            e[3] = int32_t(tok > max_tokens ? max_tokens : tok);
            e[4] = int32_t(s);
            e[5] = int32_t(len);
        }
        need_all += sum;
        tokens_all += tok_sum;
    }
    __syncthreads();
    const uint32_t there = find_free(p, need_all < p.n_pages ? need_all : p.n_pages, sh);
    // Eight lanes an entry, or a warp where entries have many tokens: each is a chain of loads, and 192 entries of a few tokens took a third of
    // the call with a warp each.
    const uint32_t width = tokens_all > 16ull * n ? 32u : 8u, lane = threadIdx.x & (width - 1u);
    for (uint32_t i = threadIdx.x / width; i < n; i += PLAN_THREADS / width) {
        const int32_t* const e = entry + APPEND_FIELDS * i;
        int32_t say = e[0];
        const uint32_t before = uint32_t(e[1]), need = uint32_t(e[2]), tok = uint32_t(e[3]);
        if (say == 0 && need && uint64_t(before) + need > there) say = ATLAS_B200_ERR_LIMIT;
        const uint32_t add = n_new[i] > 0 ? uint32_t(n_new[i]) : 0u;
        if (say == 0) {
            const uint32_t s = uint32_t(e[4]), len = uint32_t(e[5]), have = pages_of(p, len);
            int32_t* row = p.block_table + size_t(s) * p.table_stride;
            for (uint32_t k = lane; k < need; k += width) {
                const int32_t id = p.list[before + k];
                row[have + k] = id;
                p.refcount[id] = 1;
            }
            for (uint32_t k = lane; k < add; k += width) {
                const uint32_t pos = len + k, page = pos / p.block_size;
                const int32_t id = page < have ? row[page] : p.list[before + page - have];
                slot_mapping[tok + k] = uint32_t(id) < p.n_pages ? (long long)(id) * p.block_size + (pos - page * p.block_size) : -1ll;
                if (uint32_t(id) >= p.n_pages) record_status(STATUS_PAGE_OUT_OF_RANGE);
            }
            if (lane == 0) p.seq_len[s] = int32_t(len + add);
        } else {
            for (uint32_t k = lane; k < add && tok + k < max_tokens; k += width) slot_mapping[tok + k] = -1ll;
        }
        if (lane == 0 && status) status[i] = say;
    }
    for (uint64_t k = tokens_all + threadIdx.x; k < max_tokens; k += PLAN_THREADS) slot_mapping[k] = -1ll;
}

// ---- fork --------------------------------------------------------------------------------------------------------
// Entry i makes the empty sequence dst[i] a copy of src[i] as it stood before the call.
__global__ void __launch_bounds__(PLAN_THREADS) fork_plan_kernel(PagesParams p, const int32_t* src, const int32_t* dst, uint32_t n, int32_t* status) {
    __shared__ uint64_t sh[32];
    pdl_release();
    pdl_wait();
    src = pdl_after(src); dst = pdl_after(dst); p.refcount = pdl_after(p.refcount); p.block_table = pdl_after(p.block_table); p.seq_len = pdl_after(p.seq_len);
    claim_seqs(p, dst, n);
    const uint64_t room = uint64_t(p.table_stride) * p.block_size;
    uint64_t need_all = 0;
    for (uint32_t base = 0; base < n; base += PLAN_THREADS) {
        const uint32_t i = base + threadIdx.x;
        int32_t say = ATLAS_B200_ERR_DIMS, len = 0;
        if (i < n) {
            const uint32_t a = uint32_t(src[i]), b = uint32_t(dst[i]);
            if (a < p.n_seqs && b < p.n_seqs && a != b && __ldcg(p.claim + b) == int32_t(i) && p.seq_len[b] == 0 && p.seq_len[a] >= 0 && uint64_t(p.seq_len[a]) <= room) {
                say = 0;
                len = p.seq_len[a];
            }
        }
        const uint32_t need = say == 0 && uint32_t(len) % p.block_size ? 1u : 0u;
        uint64_t sum;
        const uint64_t before = need_all + block_scan(need, sh, sum);
        if (i < n) { p.entry[4 * i] = say; p.entry[4 * i + 1] = int32_t(before); p.entry[4 * i + 2] = len; }
        need_all += sum;
    }
    __syncthreads();                                                         // lengths have been read; they are written below
    const uint32_t there = find_free(p, need_all < p.n_pages ? need_all : p.n_pages, sh);
    for (uint32_t i = threadIdx.x; i < n; i += PLAN_THREADS) {
        int32_t say = p.entry[4 * i];
        const uint32_t len = uint32_t(p.entry[4 * i + 2]), before = uint32_t(p.entry[4 * i + 1]);
        int32_t fresh = -1;
        if (say == 0 && len % p.block_size) {
            if (before < there) { fresh = p.list[before]; p.refcount[fresh] = 1; }
            else say = ATLAS_B200_ERR_LIMIT;
        }
        p.entry[4 * i] = say;
        p.entry[4 * i + 3] = fresh;
        if (say == 0) p.seq_len[dst[i]] = int32_t(len);
        if (status) status[i] = say;
    }
}

// One base's bytes from page to page; a base that is not on a 16-byte boundary (which the host cannot see) is copied byte by byte.
__device__ __forceinline__ void copy_page(const PagesParams& p, uint32_t b, uint32_t to_page, uint32_t from_page, uint64_t bytes) {
    uint8_t* const base = reinterpret_cast<uint8_t*>(p.bases[b]);
    if (!base) return;
    uint8_t* const to = base + uint64_t(to_page) * p.page_bytes;
    const uint8_t* const from = base + uint64_t(from_page) * p.page_bytes;
    const uint64_t n = (reinterpret_cast<uintptr_t>(base) & 15u) ? 0 : bytes / 16;
    uint4* const d = reinterpret_cast<uint4*>(to);
    const uint4* const s = reinterpret_cast<const uint4*>(from);
    for (uint64_t at = threadIdx.x; at < n; at += 8 * COPY_THREADS) {
        uint4 v[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k)
            if (at + k * COPY_THREADS < n) v[k] = __ldcs(s + at + k * COPY_THREADS);
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k)
            if (at + k * COPY_THREADS < n) __stcs(d + at + k * COPY_THREADS, v[k]);
    }
    for (uint64_t at = n * 16 + threadIdx.x; at < bytes; at += COPY_THREADS) to[at] = from[at];
}

// CTA (x, y): entry x, bases y, y + gridDim.y, ...; y = 0 copies the row of the table too.
__global__ void __launch_bounds__(COPY_THREADS) fork_copy_kernel(PagesParams p, const int32_t* src, const int32_t* dst) {
    pdl_release();
    pdl_wait();
    p.entry = pdl_after(p.entry);
    const uint32_t i = blockIdx.x;
    if (p.entry[4 * i] != 0) return;
    const uint32_t len = uint32_t(p.entry[4 * i + 2]), full = len / p.block_size, rest = len % p.block_size;
    const int32_t* from = p.block_table + size_t(src[i]) * p.table_stride;
    const int32_t fresh = p.entry[4 * i + 3];
    if (blockIdx.y == 0) {
        int32_t* to = p.block_table + size_t(dst[i]) * p.table_stride;
        for (uint32_t k = threadIdx.x; k < full; k += COPY_THREADS) {
            const int32_t id = from[k];
            to[k] = id;
            if (uint32_t(id) < p.n_pages) atomicAdd(p.refcount + id, 1);
            else record_status(STATUS_PAGE_OUT_OF_RANGE);
        }
        if (rest && threadIdx.x == 0) to[full] = fresh;
    }
    if (!rest) return;
    const uint32_t old = uint32_t(from[full]);
    if (old >= p.n_pages) { record_status(STATUS_PAGE_OUT_OF_RANGE); return; }
    const uint64_t bytes = p.page_bytes / p.block_size * rest;
    for (uint32_t b = blockIdx.y; b < p.n_bases; b += gridDim.y) {
        copy_page(p, b, uint32_t(fresh), old, bytes);
    }
}

// ---- free --------------------------------------------------------------------------------------------------------
constexpr int FREE_THREADS = 128;
__global__ void __launch_bounds__(FREE_THREADS) free_kernel(PagesParams p, const int32_t* seqs) {
    __shared__ int32_t len_s;
    pdl_release();
    pdl_wait();
    seqs = pdl_after(seqs);
    const uint32_t s = uint32_t(seqs[blockIdx.x]);
    if (s >= p.n_seqs) { if (threadIdx.x == 0) record_status(STATUS_SEQ_OUT_OF_RANGE); return; }
    if (threadIdx.x == 0) len_s = atomicExch(p.seq_len + s, 0);              // of two entries that name a sequence one finds it
    __syncthreads();
    const int32_t len = len_s;
    if (len <= 0) return;
    const uint64_t held = (uint64_t(len) + p.block_size - 1) / p.block_size;
    const uint32_t n = uint32_t(held < p.table_stride ? held : p.table_stride);
    int32_t* row = p.block_table + size_t(s) * p.table_stride;
    for (uint32_t k = threadIdx.x; k < n; k += FREE_THREADS) {
        const int32_t id = row[k];
        row[k] = -1;
        if (uint32_t(id) >= p.n_pages) { record_status(STATUS_PAGE_OUT_OF_RANGE); continue; }
        if (atomicSub(p.refcount + id, 1) <= 0) { atomicAdd(p.refcount + id, 1); record_status(STATUS_PAGE_NOT_HELD); }
    }
}

// ---- compact -----------------------------------------------------------------------------------------------------
// With U pages in use, the k-th page in use behind the first U goes to the k-th free page among them.
__global__ void __launch_bounds__(PLAN_THREADS) compact_plan_kernel(PagesParams p, int32_t* ref_out, int32_t* page_map, int32_t* n_used) {
    __shared__ uint64_t sh[32];
    pdl_release();
    pdl_wait();
    p.refcount = pdl_after(p.refcount);
    uint32_t mine = 0;
    for (uint32_t at = threadIdx.x; at < p.n_pages; at += PLAN_THREADS) mine += p.refcount[at] > 0;
    uint64_t used;
    block_scan(mine, sh, used);
    uint64_t so_far = 0;                                                     // holes in the low half, moved pages in the high half
    for (uint32_t base = 0; base < p.n_pages; base += 4 * PLAN_THREADS) {
        const uint32_t at = base + 4 * threadIdx.x;
        int32_t ref[4];
        uint64_t count = 0;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            ref[k] = at + k < p.n_pages ? p.refcount[at + k] : 0;
            if (at + k < used && ref[k] <= 0) count += 1;
            if (at + k >= used && ref[k] > 0) count += 1ull << 32;
        }
        uint64_t sum;
        uint64_t to = so_far + block_scan(count, sh, sum);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            if (at + k >= p.n_pages) break;
            const bool hole = at + k < used && ref[k] <= 0, moved = at + k >= used && ref[k] > 0;
            if (hole) { p.list[uint32_t(to)] = int32_t(at + k); ++to; }
            if (moved) { p.list[p.n_pages - 1 - uint32_t(to >> 32)] = int32_t(at + k); to += 1ull << 32; }
            if (!moved) page_map[at + k] = ref[k] > 0 ? int32_t(at + k) : -1;
            if (!hole && !moved) ref_out[at + k] = ref[k];
        }
        so_far += sum;
    }
    __syncthreads();
    const uint32_t moves = uint32_t(so_far);                                 // as many holes as moved pages
    for (uint32_t k = threadIdx.x; k < moves; k += PLAN_THREADS) {
        const int32_t from = p.list[p.n_pages - 1 - k], to = p.list[k];
        page_map[from] = to;
        const int32_t held = p.refcount[from];
        ref_out[to] = held;
        ref_out[from] = 0;
    }
    if (threadIdx.x == 0) { *n_used = int32_t(used); p.count[0] = int32_t(moves); }
}

__global__ void __launch_bounds__(COPY_THREADS) compact_move_kernel(PagesParams p, const int32_t* page_map, int32_t* table_out) {
    pdl_release();
    pdl_wait();
    p.list = pdl_after(p.list);
    const uint64_t moves = uint32_t(p.count[0]), jobs = moves * p.n_bases;
    for (uint64_t j = blockIdx.x; j < jobs; j += gridDim.x) {
        const uint32_t k = uint32_t(j / p.n_bases), b = uint32_t(j % p.n_bases);
        copy_page(p, b, uint32_t(p.list[k]), uint32_t(p.list[p.n_pages - 1 - k]), p.page_bytes);
    }
    // the tables, by the CTAs from the last one on, which have the fewest copies
    for (uint32_t s = gridDim.x - 1 - blockIdx.x; s < p.n_seqs; s += gridDim.x) {
        const int32_t len = p.seq_len[s];
        const uint64_t held = len > 0 ? (uint64_t(len) + p.block_size - 1) / p.block_size : 0;
        const size_t row = size_t(s) * p.table_stride;
        for (uint32_t k = threadIdx.x; k < p.table_stride; k += COPY_THREADS) {
            const int32_t id = p.block_table[row + k];
            if (k < held && uint32_t(id) >= p.n_pages) record_status(STATUS_PAGE_OUT_OF_RANGE);
            table_out[row + k] = k < held && uint32_t(id) < p.n_pages ? page_map[id] : id;
        }
    }
}

}  // namespace pages
}  // namespace atlas
