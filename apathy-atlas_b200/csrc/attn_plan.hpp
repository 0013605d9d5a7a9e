// How the attention over the paged cache is cut into pieces of equal work, in plain C++ so that it is checked on the CPU.
//
// Of one sequence and one KV head, the chunk's rows are its new tokens times the `group` query heads that share the KV head: row r is
// token r / group, head r % group of them.  `block_rows` rows make a block; a block reads the keys its last row sees, in tiles of
// `tile_keys`.  An item is one (sequence, block, KV head).  All items' tiles in a row (sequence, block, KV head, tile; the last fastest)
// are the line that CTAs cut into contiguous ranges of equal length, whatever the sequences' lengths: a range may begin and end inside
// an item, whose pieces are joined afterwards.  What an item costs besides its tiles (fetching Q, writing the output) stands in the line
// as `extra` places ahead of its first tile.  A cut among those is none: the item belongs to the range behind it.
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifndef ATLAS_HD
#ifdef __CUDACC__
#define ATLAS_HD __host__ __device__
#else
#define ATLAS_HD
#endif
#endif

namespace atlas {

// A quotient, in 32 bits where both numbers have no more: a GPU divides those in a tenth of the time, and the numbers of a plan, which
// every CTA works out before it can ask for its first key, nearly always have.
ATLAS_HD inline uint64_t attn_quotient(uint64_t a, uint64_t b) { return ((a | b) >> 32) == 0 ? uint64_t(uint32_t(a) / uint32_t(b)) : a / b; }

// sum of floor((a i + b) / m) over i = 0 .. n - 1, by Euclid's algorithm on (a, m)
ATLAS_HD inline uint64_t floor_sum(uint64_t n, uint64_t m, uint64_t a, uint64_t b) {
    uint64_t sum = 0;
    while (n > 0) {
        if (a >= m) { const uint64_t q = attn_quotient(a, m); sum += q * (n * (n - 1) / 2); a -= q * m; }
        if (b >= m) { const uint64_t q = attn_quotient(b, m); sum += q * n; b -= q * m; }
        const uint64_t last = a * n + b;
        if (last < m) break;
        n = attn_quotient(last, m);
        b = last - n * m;
        const uint64_t t = m;
        m = a;
        a = t;
    }
    return sum;
}

// One sequence's blocks.  Without new tokens it has none; with fewer cached tokens than new ones (the first rows see nothing) all of
// its blocks count as if they saw the whole cache.
struct AttnSeq {
    uint32_t q_len, kv_len, blocks, whole;      // whole: tiles of the cached tokens, one at least
    uint32_t group, block_rows, tile_keys, extra;
    ATLAS_HD AttnSeq(uint32_t q, uint32_t kv, uint32_t g, uint32_t rows, uint32_t keys, uint32_t more)
        : q_len(q), kv_len(kv), group(g), block_rows(rows), tile_keys(keys), extra(more) {
        blocks = uint32_t(attn_quotient(uint64_t(q) * g + rows - 1, rows));
        whole = kv ? (kv - 1) / keys + 1 : 1;
    }
    // the last row of block b is row (b + 1) rows - 1, token floor of it / group; it sees kv_len - q_len + that token + 1 keys
    ATLAS_HD uint32_t tiles(uint32_t b) const {
        if (kv_len < q_len || b + 1 >= blocks) return whole;
        const uint64_t keys_less_1 = uint64_t(kv_len - q_len) + tile_keys;
        const uint64_t t = attn_quotient(uint64_t(block_rows) * b + block_rows - 1 + uint64_t(group) * keys_less_1, uint64_t(group) * tile_keys);
        return t < whole ? uint32_t(t) : whole;
    }
    // places of the blocks before b, of one KV head
    ATLAS_HD uint64_t before(uint32_t b) const {
        if (b == 0 || blocks == 0) return 0;
        if (blocks == 1) return uint64_t(whole) + extra;
        const uint32_t n = b < blocks ? b : blocks - 1;                                   // by the formula
        uint64_t sum = kv_len < q_len ? uint64_t(whole) * n
                                      : floor_sum(n, uint64_t(group) * tile_keys, block_rows, block_rows - 1 + uint64_t(group) * (uint64_t(kv_len - q_len) + tile_keys));
        return (b < blocks ? sum : sum + whole) + uint64_t(b) * extra;
    }
    ATLAS_HD uint64_t total(uint32_t kv_heads) const { return before(blocks) * kv_heads; }
};

struct AttnPlace {
    uint32_t block, head, place, tiles;         // place within the item, which has extra + tiles of them
};
// where place x lies, known to be in a block
ATLAS_HD inline AttnPlace attn_place_in_block(const AttnSeq& s, uint32_t kv_heads, uint64_t x, uint32_t block) {
    AttnPlace p;
    p.block = block;
    p.tiles = s.tiles(block);
    const uint64_t in_block = x - s.before(block) * kv_heads;
    p.head = uint32_t(attn_quotient(in_block, s.extra + p.tiles));
    p.place = uint32_t(in_block - uint64_t(p.head) * (s.extra + p.tiles));
    return p;
}
// where place x of a sequence's part of the line lies, x < total(kv_heads)
ATLAS_HD inline AttnPlace attn_locate(const AttnSeq& s, uint32_t kv_heads, uint64_t x) {
    uint32_t lo = 0, hi = s.blocks - 1;
    while (lo < hi) {                                                                     // the last block that begins at or before x
        const uint32_t mid = (lo + hi + 1) / 2;
        if (s.before(mid) * kv_heads <= x) lo = mid;
        else hi = mid - 1;
    }
    return attn_place_in_block(s, kv_heads, x, lo);
}

// The next item of a sequence's part of the line; false behind the last.
ATLAS_HD inline bool attn_next(const AttnSeq& s, uint32_t kv_heads, AttnPlace& p) {
    p.place = 0;
    if (++p.head < kv_heads) return true;
    p.head = 0;
    if (++p.block >= s.blocks) return false;
    p.tiles = s.tiles(p.block);
    return true;
}

// Range c of `ranges` over a line of `total` places begins here; range_of: the one that place x belongs to.
ATLAS_HD inline uint64_t attn_range_begin(uint64_t total, uint32_t ranges, uint32_t c) {
    const uint64_t each = attn_quotient(total, ranges), more = total - each * ranges;     // the first `more` are one longer
    return each * c + (c < more ? c : more);
}
ATLAS_HD inline uint32_t attn_range_of(uint64_t total, uint32_t ranges, uint64_t x) {
    const uint64_t each = attn_quotient(total, ranges), more = total - each * ranges;
    const uint64_t longer = more * (each + 1);
    return x < longer ? uint32_t(attn_quotient(x, each + 1)) : uint32_t(more + attn_quotient(x - longer, each));
}
// how many of the `ctas` CTAs take part where each is to have `least` places at least
ATLAS_HD inline uint32_t attn_ranges(uint64_t total, uint32_t ctas, uint32_t least) {
    const uint64_t n = attn_quotient(total + least - 1, least);
    return n < 1 ? 1u : n < ctas ? uint32_t(n) : ctas;
}

}  // namespace atlas
