// Attention of the new tokens of a batch of sequences over their paged K/V cache: what the kernels share.
//
//   o[t, h] = sum_j p_j v[j, h / group],   p = softmax_j( scale * q[t, h] . k[j, h / group] ),   j <= kv_len - q_len + (t - first token)
//
// with the running maximum and sum of a softmax held in FP32: of each piece of the keys a kernel has M (largest score, in units of
// log 2), L = sum 2^(s - M) and O = sum 2^(s - M) v; two pieces join as M = max, L = L1 2^(M1 - M) + L2 2^(M2 - M), O likewise.
// A row that sees no key has L = 0 and gives zeros, and -inf as its logarithm.  (Any M does, as long as the weights stay within their type:
// over E4M3 caches, whose weights are FP16, it is 2^7 below the largest, see ATTN_UP.)
//
// The line of tiles of all items (attn_plan.hpp) is cut into one range a CTA.  An item that lies in one range is written at once; the
// pieces of one that does not go to scratch, two slots a CTA (the item its range begins in, the item its range ends in), and
// attn_join_kernel adds them in the order of their keys: the same call gives the same bits.
#pragma once

#include <cstdint>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "attn_plan.hpp"
#include "common.cuh"

namespace atlas {

constexpr float ATTN_LOG2E = 1.4426950408889634f, ATTN_LN2 = 0.6931471805599453f;

struct AttnParams {
    const uint16_t* q;            // first column of row 0, rows q_row_stride elements apart
    uint16_t* out;
    float* lse;                   // [n_tokens, q_heads], or null
    const uint8_t* k_cache;       // [n_pages, block_size, kv_heads, head_dim]
    const uint8_t* v_cache;
    const int32_t* block_table;   // [n_seqs, table_stride]
    const int32_t* cu_q;          // [n_seqs + 1]
    const int32_t* kv_len;        // [n_seqs]
    struct AttnCut* cuts;         // [ctas] where each range begins (see AttnCut)
    float* parts;                 // two slots a range of block_rows rows: O, then M and L (see attn_part_floats)
    uint32_t n_seqs, n_tokens, n_pages, table_stride, q_heads, kv_heads, head_dim, block_size, group, q_row_stride, out_row_stride;
    uint32_t ctas, least_tiles;   // ranges: at most `ctas`, of `least_tiles` tiles each at least
    uint32_t by_item;             // every CTA (or cluster) takes whole items: no pieces in scratch
    uint32_t cluster_log2;        // by_item: an item is a cluster's of 2^this CTAs, each with a share of its tiles
    AttnShape shape;              // of the kernel's blocks and tiles
    AttnDivisor page_div, group_div;
    float scale, k_scale, v_scale;
};

__host__ __device__ constexpr size_t attn_part_floats(uint32_t block_rows, uint32_t dim) { return size_t(block_rows) * dim + 2 * block_rows; }

struct AttnSeqAt {
    uint32_t row0, q_len, kv_len;
};
// A sequence as its tables have it, held to what the buffers hold.
__device__ __forceinline__ AttnSeqAt attn_seq(const AttnParams& p, uint32_t s) {
    const int32_t a = p.cu_q[s], b = p.cu_q[s + 1], n = p.kv_len[s];
    AttnSeqAt r;
    r.row0 = a < 0 ? 0u : min(uint32_t(a), p.n_tokens);
    const uint32_t end = b < 0 ? 0u : min(uint32_t(b), p.n_tokens);
    r.q_len = end > r.row0 ? end - r.row0 : 0u;
    const uint64_t room = uint64_t(p.table_stride) * p.block_size;
    r.kv_len = n < 0 ? 0u : (uint64_t(n) > room ? uint32_t(room) : uint32_t(n));
    if (n > 0 && uint64_t(n) > room && r.q_len) record_status(STATUS_CACHE_LENGTH);   // (a sequence without new tokens is skipped, whatever its length says)
    return r;
}

// What the join has to know of the item that a range begins inside, written by the range's CTA, which has it at hand.
struct AttnCut {
    uint32_t pieces;              // of the item, on this range and the next ones and the one before; 0: no item is cut here for the first time
    uint32_t seq, block, head;
};

// FP16 holds nothing below 2^-24, so beside a largest weight of 1 a weight below 2^-25 would count in the sum and not in the output: over 2^18
// keys at 2^-25.4 of the largest, 2^-7 of it.  With M lower by ATTN_UP the largest weight is 2^7 and that border 2^-32.  (No more than 7: scores
// are FP32, whose steps are 16 from 2^27 on.  M rounded to such steps keeps within 2^8 of the largest score's weight, itself off by 2^8 there.)
constexpr float ATTN_UP = 7.0f;
// M for a largest product `top` of a row and its factor
template <bool FP8> __device__ __forceinline__ float attn_base(float top, float c) {
    if constexpr (FP8) return fmaf(top, c, -ATTN_UP);
    else return top * c;
}

// The scores' factor must not come to zero: zero times a masked place's -inf is a NaN.  From here down all scores are equal.
__device__ __forceinline__ float attn_factor(float c) { return fmaxf(c, 1.1754944e-38f); }

// 2^x by the special-function unit; off by 2^-22 of the value at most, 0 below 2^-126
__device__ __forceinline__ float attn_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// How many keys new token i of a sequence sees.
__device__ __forceinline__ uint32_t attn_row_keys(const AttnSeqAt& s, uint32_t i) {
    const uint64_t n = uint64_t(s.kv_len) + i + 1;
    return n <= s.q_len ? 0u : uint32_t(n - s.q_len);
}

// Where a CTA's range of the line begins: worked out by one warp, while the others have nothing to do yet (all of them going through the
// same divisions took twice as long), and left in shared memory.
struct AttnStart {
    uint64_t left;                // places of the range; 0: there is none
    AttnPlace at;
    AttnSeqAt sq;
    uint32_t seq;
};
__device__ __forceinline__ uint64_t attn_seq_places(const AttnParams& p, uint32_t s) {
    const AttnSeqAt q = attn_seq(p, s);
    const AttnSeq a(q.q_len, q.kv_len, p.shape);
    return p.by_item ? uint64_t(a.blocks) * p.kv_heads : a.total(p.kv_heads);
}
__device__ __forceinline__ uint64_t attn_warp_scan(uint64_t mine) {          // inclusive
    const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
    for (uint32_t o = 1; o < 32; o <<= 1) {
        const uint64_t v = __shfl_up_sync(0xFFFFFFFFu, mine, o);
        if (lane >= o) mine += v;
    }
    return mine;
}
// By one warp: the place `begin` of the sequence's part of the line, whose first place is seq_begin; and a note of the cut there.
__device__ __forceinline__ void attn_begin_at(const AttnParams& p, const AttnRanges& ranges, uint64_t begin, uint64_t end, uint32_t seq, uint64_t seq_begin, AttnStart* start) {
    const uint32_t lane = threadIdx.x & 31u, c = blockIdx.x >> p.cluster_log2;
    const AttnSeqAt sq = attn_seq(p, seq);
    const AttnSeq plan(sq.q_len, sq.kv_len, p.shape);
    const uint64_t x = begin - seq_begin;
    AttnPlace at;
    if (p.by_item) {
        at.block = uint32_t(attn_quotient(x, p.kv_heads));
        at.head = uint32_t(x - uint64_t(at.block) * p.kv_heads);
        at.place = 0;
        at.tiles = plan.tiles(at.block);
    } else {
        at = attn_locate(plan, p.kv_heads, x, [lane](auto holds) { return uint32_t(__popc(__ballot_sync(0xFFFFFFFFu, holds(lane)))); });
    }
    if (lane != 0) return;
    start->left = end - begin;
    start->at = at;
    start->sq = sq;
    start->seq = seq;
    if (p.by_item) return;
    p.cuts[c] = AttnCut{attn_cut_pieces(ranges, c, begin, at, p.shape.extra), seq, at.block, at.head};
}
// By all THREADS threads of a CTA; `sh`: THREADS / 32 words of 64 bits.  Ends with a barrier.
constexpr uint32_t ATTN_WARP_SEQS = 256;
template <int THREADS>
__device__ __forceinline__ void attn_begin(const AttnParams& p, uint64_t* sh, AttnStart* start) {
    constexpr uint32_t WARPS = THREADS / 32;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, c = blockIdx.x >> p.cluster_log2;
    const bool few = p.n_seqs <= ATTN_WARP_SEQS;                             // one warp sums up the sequences too
    if (!few || warp == 0) {
        const uint32_t by = few ? 32u : uint32_t(THREADS), each = (p.n_seqs + by - 1) / by, s0 = min(tid * each, p.n_seqs), s1 = min(s0 + each, p.n_seqs);
        uint64_t mine = 0;
        for (uint32_t s = s0; s < s1; ++s) mine += attn_seq_places(p, s);
        uint64_t upto = attn_warp_scan(mine), total = __shfl_sync(0xFFFFFFFFu, upto, 31);
        if (!few) {
            if (lane == 31u) sh[warp] = upto;
            __syncthreads();
            total = 0;
            for (uint32_t w = 0; w < WARPS; ++w) {
                if (w < warp) upto += sh[w];
                total += sh[w];
            }
        }
        const AttnRanges ranges(total, p.ctas, p.least_tiles);
        const uint64_t begin = c < ranges.n ? ranges.begin(c) : 0, end = c < ranges.n ? ranges.begin(c + 1) : 0;
        if (begin == end) {
            if (tid == 0) {
                start->left = 0;
                if (!p.by_item) p.cuts[c].pieces = 0;                        // more CTAs than ranges
            }
        } else {
            const bool owns = mine && begin < upto && begin >= upto - mine;  // one lane of one warp
            const uint32_t who = __ballot_sync(0xFFFFFFFFu, owns);
            if (who) {
                uint32_t seq = s0;
                uint64_t at = upto - mine;
                if (owns && s1 - s0 > 1)
                    for (uint64_t k; seq + 1 < s1 && begin >= at + (k = attn_seq_places(p, seq)); ++seq) at += k;
                const uint32_t lane_of = __ffs(who) - 1u;
                attn_begin_at(p, ranges, begin, end, __shfl_sync(0xFFFFFFFFu, seq, lane_of), __shfl_sync(0xFFFFFFFFu, at, lane_of), start);
            }
        }
    }
    __syncthreads();
}

// The items of one CTA's range, one after the other; every thread walks by itself.
struct AttnWalk {
    AttnSeqAt sq;
    AttnPlace at;                 // of the item; its piece is tiles t0 .. t1 - 1
    uint32_t seq, t0, t1;

    __device__ __forceinline__ AttnWalk(const AttnStart& s) : sq(s.sq), at(s.at), seq(s.seq), t0(0), t1(0), left_(s.left), fresh_(true) {}
    __device__ __forceinline__ AttnSeq plan(const AttnParams& p) const { return AttnSeq(sq.q_len, sq.kv_len, p.shape); }
    __device__ __forceinline__ bool next(const AttnParams& p) {
        if (!left_) return false;
        if (!fresh_ && !attn_next(plan(p), p.kv_heads, at)) {
            do { ++seq; sq = attn_seq(p, seq); } while (sq.q_len == 0);      // (the range ends at a sequence that has places)
            at.block = at.head = at.place = 0;
            at.tiles = plan(p).tiles(0);
        }
        fresh_ = false;
        if (p.by_item) {
            t0 = 0;
            t1 = at.tiles;
            --left_;
            return true;
        }
        const uint32_t there = p.shape.extra + at.tiles, end = there - at.place <= left_ ? there : at.place + uint32_t(left_);
        left_ -= end - at.place;
        t0 = at.place > p.shape.extra ? at.place - p.shape.extra : 0u;
        t1 = end > p.shape.extra ? end - p.shape.extra : 0u;
        return t1 != 0u;                                                     // (a range that ends ahead of an item's first tile)
    }
    __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == at.tiles; }

private:
    uint64_t left_;
    bool fresh_;
};

// Row `pos` of a sequence in the cache seen as [pages * block_size, kv_heads, head_dim]; -1 and a record where the table names no page.
__device__ __forceinline__ int32_t attn_cache_row(const AttnParams& p, const int32_t* table, uint32_t pos) {
    const uint32_t page = attn_div(pos, p.page_div), id = uint32_t(table[page]);
    if (id >= p.n_pages) { record_status(STATUS_PAGE_OUT_OF_RANGE); return -1; }
    return int32_t(id * p.block_size + (pos - page * p.block_size));
}

__device__ __forceinline__ float attn_e4m3(uint8_t b) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3))); }

// Logarithm of a row's sum of exponentials from its M and L.
__device__ __forceinline__ float attn_lse(float m, float l) { return l == 0.0f ? -INFINITY : (m + log2f(l)) * ATTN_LN2; }

// The kernels multiply masked places with zeros, and zero times an infinity or a NaN in the values of a later token is a NaN.  So a row
// that came out not finite is computed once more, by one warp from its own keys alone, where such values stand among the keys that its
// block reads and it does not see: ATTN_MASKED_MOST behind its own at most (256 rows of a block, and what is left of a tile of 128).
// Where there are none the row is what its formula gives.  32 keys at a time: a lane has a key's score, then the warp the key's values.
constexpr uint32_t ATTN_MASKED_MOST = 384;

__device__ __forceinline__ float attn_cache_value(const uint8_t* cache, bool fp8, size_t at) {
    return fp8 ? attn_e4m3(cache[at]) : __uint_as_float(uint32_t(reinterpret_cast<const uint16_t*>(cache)[at]) << 16);
}
// Whether a value of keys from .. to - 1 is not finite; by one warp.
static __device__ __noinline__ bool attn_odd_values(const AttnParams& p, bool fp8, uint32_t seq, uint32_t kv_head, uint32_t from, uint32_t to) {
    const uint32_t lane = threadIdx.x & 31u, D = p.head_dim;
    const int32_t* table = p.block_table + size_t(seq) * p.table_stride;
    bool odd = false;
    for (uint32_t j0 = from; j0 < to; j0 += 32) {
        const int32_t row = j0 + lane < to ? attn_cache_row(p, table, j0 + lane) : -1;
        for (uint32_t d = lane; d < D; d += 32)
#pragma unroll 8
            for (uint32_t k = 0; k < 32; ++k) {
                const int32_t r = __shfl_sync(0xFFFFFFFFu, row, k);
                if (r >= 0) odd |= !isfinite(attn_cache_value(p.v_cache, fp8, (size_t(r) * p.kv_heads + kv_head) * D + d));
            }
        if (__any_sync(0xFFFFFFFFu, odd)) return true;
    }
    return false;
}
template <bool fp8>
__device__ __noinline__ void attn_row_again(const AttnParams& p, uint32_t seq, uint32_t token, uint32_t head, uint32_t keys, uint32_t kv_len) {
    const uint32_t lane = threadIdx.x & 31u, D = p.head_dim, kv_head = head / p.group;
    if (!attn_odd_values(p, fp8, seq, kv_head, keys, min(kv_len, keys + ATTN_MASKED_MOST))) return;
    const int32_t* table = p.block_table + size_t(seq) * p.table_stride;
    const uint32_t* q = reinterpret_cast<const uint32_t*>(p.q + size_t(token) * p.q_row_stride + size_t(head) * D);
    constexpr uint32_t size = fp8 ? 1 : 2, AT_ONCE = 4;
    float o[8] = {}, m = -INFINITY, l = 0.0f;
    const float c = attn_factor(p.scale * p.k_scale * ATTN_LOG2E);
    for (uint32_t j0 = 0; j0 < keys; j0 += 32) {
        const uint32_t n = min(keys - j0, 32u);
        const int32_t row = lane < n ? attn_cache_row(p, table, j0 + lane) : -1;
        float s = 0.0f;
        if (row >= 0) {
            const uint4* k_row = reinterpret_cast<const uint4*>(p.k_cache + (size_t(row) * p.kv_heads + kv_head) * D * size);
            const uint32_t chunks = D * size / 16;
            for (uint32_t c0 = 0; c0 < chunks; c0 += AT_ONCE) {
                uint4 v[AT_ONCE];
#pragma unroll
                for (uint32_t i = 0; i < AT_ONCE; ++i) v[i] = c0 + i < chunks ? k_row[c0 + i] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (uint32_t i = 0; i < AT_ONCE; ++i) {
                    if (c0 + i >= chunks) break;
                    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                    for (uint32_t e = 0; e < 8 / size; ++e) {
                        const uint32_t qq = q[8 / size * (c0 + i) + e];
                        if constexpr (fp8) {
                            const uint32_t two = w[e >> 1] >> (16 * (e & 1));
                            s = fmaf(bf16_lo(qq), attn_e4m3(uint8_t(two)), s);
                            s = fmaf(bf16_hi(qq), attn_e4m3(uint8_t(two >> 8)), s);
                        } else {
                            s = fmaf(bf16_lo(qq), bf16_lo(w[e]), s);
                            s = fmaf(bf16_hi(qq), bf16_hi(w[e]), s);
                        }
                    }
                }
            }
        }
        s = lane < n ? s * c : -INFINITY;
        float top = fmaxf(m, s);
        for (uint32_t x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
        const float base = top == -INFINITY ? 0.0f : top, keep = exp2f(m - base), w = exp2f(s - base);
        l = l * keep + w;
        for (uint32_t i = 0; i < 8; ++i) o[i] *= keep;
        for (uint32_t k0 = 0; k0 < n; k0 += AT_ONCE) {                       // (lanes behind n have no row and no weight)
            float v[AT_ONCE][8], w_k[AT_ONCE];
#pragma unroll
            for (uint32_t k = 0; k < AT_ONCE; ++k) {
                const int32_t r = __shfl_sync(0xFFFFFFFFu, row, k0 + k);
                w_k[k] = __shfl_sync(0xFFFFFFFFu, w, k0 + k);
                const size_t at = (size_t(r < 0 ? 0 : r) * p.kv_heads + kv_head) * D;
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) v[k][i] = r >= 0 && lane + 32u * i < D ? attn_cache_value(p.v_cache, fp8, at + lane + 32u * i) : 0.0f;
            }
#pragma unroll
            for (uint32_t k = 0; k < AT_ONCE; ++k)
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) o[i] += w_k[k] * v[k][i];
        }
        m = top;
    }
    for (uint32_t x = 16; x; x >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, x);
    const float f = l == 0.0f ? 0.0f : p.v_scale / l;
    if (p.lse && lane == 0) p.lse[size_t(token) * p.q_heads + head] = attn_lse(m, l);
    for (uint32_t i = 0; i < 8; ++i)
        if (lane + 32u * i < D) p.out[size_t(token) * p.out_row_stride + size_t(head) * D + lane + 32u * i] = f32_to_bf16_bits(l == 0.0f ? 0.0f : o[i] * f);
}

// ------------------------------------------------------------------------------------------------------------------
// Joins the pieces of items that were cut.  CTA (c, y) looks at the cut between ranges c and c + 1; the first cut of an item joins it.  A
// piece's slot: 2 c for the item that range c begins inside, 2 c + 1 for one that begins in range c and goes on.
//
// What it costs is latency (where the item was cut, its lengths, M and L, then O), so a CTA has all its loads of a kind in flight: up to
// ATTN_JOIN_FEW pieces it takes 32 rows, a warp works out their weights, then all warps go over the rows' channels; beyond (few sequences
// over a long cache: as many pieces as CTAs) it takes a row at a time, whose pieces the warps share and add in the order of the warps.
// (With the item's place worked out here, from the lengths, the join took 50 us of the 280 of 512 tokens over 32768; a row at a time to a
// warp, 25.)
// ------------------------------------------------------------------------------------------------------------------
constexpr int ATTN_JOIN_WARPS = 8, ATTN_JOIN_THREADS = 32 * ATTN_JOIN_WARPS;
constexpr uint32_t ATTN_JOIN_FEW = 8, ATTN_JOIN_ROWS = 32;
constexpr uint32_t ATTN_JOIN_Y = 8;                                          // grid y: 8 x 32 rows cover the largest block

// N channels of a row from channel `ch` on; true if one is not finite
template <int N>
__device__ __forceinline__ bool attn_store(const AttnParams& p, uint32_t token, uint32_t head, uint32_t ch, const float (&o)[N], float l) {
    const float inv = l == 0.0f ? 0.0f : p.v_scale / l;
    uint16_t* const to = p.out + size_t(token) * p.out_row_stride + size_t(head) * p.head_dim + ch;
    if (ch >= p.head_dim) return false;                                      // (head_dim is a multiple of 32, and N divides it)
    bool odd = false;
    uint32_t y[N / 2];
#pragma unroll
    for (int k = 0; k < N; k += 2) {
        const float a = l == 0.0f ? 0.0f : o[k] * inv, b = l == 0.0f ? 0.0f : o[k + 1] * inv;
        odd |= !isfinite(a) || !isfinite(b);
        y[k / 2] = pack_bf16x2(a, b);
    }
    if ((reinterpret_cast<uintptr_t>(to) & (2u * N - 1u)) == 0u) {
        if constexpr (N == 2) *reinterpret_cast<uint32_t*>(to) = y[0];
        if constexpr (N == 4) *reinterpret_cast<uint2*>(to) = make_uint2(y[0], y[1]);
        if constexpr (N == 8) *reinterpret_cast<uint4*>(to) = make_uint4(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) to[k] = uint16_t(y[k >> 1] >> (16 * (k & 1)));
    }
    return odd;
}

template <int ROWS, int DP, bool FP8>
__global__ void __launch_bounds__(ATTN_JOIN_THREADS, 4) attn_join_kernel(const __grid_constant__ AttnParams p) {
    __shared__ float o_s[ATTN_JOIN_WARPS][DP], w_s[ATTN_JOIN_FEW][ATTN_JOIN_ROWS], l_s[ATTN_JOIN_ROWS];
    __shared__ uint32_t odd_s;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) odd_s = 0;
    pdl_wait();
    pdl_release();
    const uint32_t c = blockIdx.x + 1;
    const AttnCut cut = p.cuts[c];
    if (cut.pieces == 0) return;
    const AttnSeqAt sq = attn_seq(p, cut.seq);
    const uint32_t rows = min(uint32_t(ROWS), sq.q_len * p.group - cut.block * ROWS);
    const size_t part = attn_part_floats(ROWS, DP);
    const float* const first = p.parts + part * (2 * size_t(c - 1) + 1);     // piece 0; piece i > 0 lies in slot 2 (c - 1 + i)
    auto piece = [&](uint32_t i) { return i == 0 ? first : p.parts + part * (2 * size_t(c - 1 + i)); };
    auto place = [&](uint32_t r, uint32_t& in_seq, uint32_t& token, uint32_t& head) {
        const uint32_t row = cut.block * ROWS + r;
        in_seq = attn_div(row, p.group_div);
        token = sq.row0 + in_seq;
        head = cut.head * p.group + row - in_seq * p.group;
    };
    uint32_t in_seq, token, head;
    if (cut.pieces <= ATTN_JOIN_FEW) {
        const uint32_t r0 = blockIdx.y * ATTN_JOIN_ROWS;
        if (r0 >= rows) return;
        const uint32_t n_rows = min(rows - r0, ATTN_JOIN_ROWS);
        if (warp == 0) {
            const uint32_t r = r0 + min(lane, n_rows - 1u);
            float m[ATTN_JOIN_FEW], l_i[ATTN_JOIN_FEW], top = -INFINITY, l = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < ATTN_JOIN_FEW; ++i) {
                const float* s = piece(min(i, cut.pieces - 1u)) + size_t(ROWS) * DP + r;
                m[i] = i < cut.pieces ? s[0] : -INFINITY;
                l_i[i] = i < cut.pieces ? s[ROWS] : 0.0f;
                top = fmaxf(top, m[i]);
            }
            const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (uint32_t i = 0; i < ATTN_JOIN_FEW; ++i) {
                const float w = exp2f(m[i] - base);
                l += w * l_i[i];
                w_s[i][lane] = w;
            }
            l_s[lane] = l;
            place(r, in_seq, token, head);
            if (p.lse && lane < n_rows) p.lse[size_t(token) * p.q_heads + head] = attn_lse(top, l);
        }
        __syncthreads();
        constexpr uint32_t LANES = DP / 4, AT_ONCE = ATTN_JOIN_THREADS / LANES;   // four channels a lane
        const uint32_t ch = (threadIdx.x % LANES) * 4u;
#pragma unroll 4
        for (uint32_t k = threadIdx.x / LANES; k < n_rows; k += AT_ONCE) {
            float o[4] = {};
#pragma unroll 2
            for (uint32_t i = 0; i < cut.pieces; ++i) {
                const float4 v = *reinterpret_cast<const float4*>(piece(i) + size_t(r0 + k) * DP + ch);
                const float w = w_s[i][k];
                o[0] += w * v.x; o[1] += w * v.y; o[2] += w * v.z; o[3] += w * v.w;
            }
            place(r0 + k, in_seq, token, head);
            if (attn_store<4>(p, token, head, ch, o, l_s[k])) atomicOr(&odd_s, 1u << k);
        }
        __syncthreads();
        for (uint32_t k = warp; k < n_rows; k += ATTN_JOIN_WARPS)
            if ((odd_s >> k) & 1u) {
                place(r0 + k, in_seq, token, head);
                attn_row_again<FP8>(p, cut.seq, token, head, attn_row_keys(sq, in_seq), sq.kv_len);
            }
        return;
    }
    if (blockIdx.y >= rows) return;                                          // (the barriers that odd_s needs are in the loop)
    constexpr int V = DP / 32;                                               // channels of a lane, side by side
    for (uint32_t r = blockIdx.y; r < rows; r += ATTN_JOIN_Y) {
        float m = -INFINITY, l = 0.0f;
        for (uint32_t i = lane; i < cut.pieces; i += 32) m = fmaxf(m, piece(i)[size_t(ROWS) * DP + r]);
        for (uint32_t x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, x));
        const float base = m == -INFINITY ? 0.0f : m;
        float o[V] = {};
        for (uint32_t i0 = 0; i0 < cut.pieces; i0 += 32) {                   // lane l: the weight of piece i0 + l
            float w_mine = 0.0f;
            if (i0 + lane < cut.pieces) {
                const float* s = piece(i0 + lane) + size_t(ROWS) * DP;
                w_mine = exp2f(s[r] - base);
                l += w_mine * s[ROWS + r];
            }
            const uint32_t n = min(cut.pieces - i0, 32u);
#pragma unroll 4
            for (uint32_t i = warp; i < n; i += ATTN_JOIN_WARPS) {
                const float w = __shfl_sync(0xFFFFFFFFu, w_mine, i);
                const float* s = piece(i0 + i) + size_t(r) * DP + lane * V;
                float v[V];
                if constexpr (V == 2) *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(s);
                else
#pragma unroll
                    for (int k = 0; k < V; k += 4) *reinterpret_cast<float4*>(v + k) = *reinterpret_cast<const float4*>(s + k);
#pragma unroll
                for (int k = 0; k < V; ++k) o[k] += w * v[k];
            }
        }
        for (uint32_t x = 16; x; x >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, x);
#pragma unroll
        for (int k = 0; k < V; ++k) o_s[warp][lane * V + k] = o[k];
        __syncthreads();
        if (warp == 0) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                o[k] = o_s[0][lane * V + k];
                for (int w = 1; w < ATTN_JOIN_WARPS; ++w) o[k] += o_s[w][lane * V + k];
            }
            place(r, in_seq, token, head);
            const bool odd = attn_store<V>(p, token, head, lane * V, o, l);
            if (p.lse && lane == 0) p.lse[size_t(token) * p.q_heads + head] = attn_lse(m, l);
            if (__any_sync(0xFFFFFFFFu, odd) && lane == 0) odd_s |= 1u << (r / ATTN_JOIN_Y);
        }
        __syncthreads();
    }
    for (uint32_t k = warp; blockIdx.y + k * ATTN_JOIN_Y < rows; k += ATTN_JOIN_WARPS)
        if ((odd_s >> k) & 1u) {
            place(blockIdx.y + k * ATTN_JOIN_Y, in_seq, token, head);
            attn_row_again<FP8>(p, cut.seq, token, head, attn_row_keys(sq, in_seq), sq.kv_len);
        }
}

}  // namespace atlas
