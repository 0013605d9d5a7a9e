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

// Quotients by a number that the host knows: a product with the rounded-up reciprocal, exact for numbers below 2^31
// (mul d = 2^(31 + shift) + e with e < d <= 2^shift, so x e < 2^(31 + shift)).
struct AttnDivisor {
    uint32_t d, mul, shift;
};
ATLAS_HD inline AttnDivisor attn_divisor(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    return AttnDivisor{d, uint32_t(((1ull << (31 + s)) + d - 1) / d), s};
}
ATLAS_HD inline uint32_t attn_div(uint32_t x, const AttnDivisor& v) { return uint32_t((uint64_t(x) * v.mul) >> (31 + v.shift)); }
// Others: in 32 bits where both numbers have no more, which a GPU divides in a tenth of the time.
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

// What is the same for all sequences of a call.  With R = 2^rows_log2 rows of a block and group * 2^keys_log2 = K: the tiles of block b are
// floor((R b + c) / K), c from the sequence.  Where K = P R that is floor((b + floor(c / R)) / P), and the sum over blocks has a closed
// form with one quotient by P, which the host knows; otherwise (an odd group of three or more over blocks of more rows than a tile has keys,
// or numbers beyond 31 bits) it is floor_sum.  Every CTA works out where its range begins before it can ask for its first key: 9000
// cycles by floor_sum.
struct AttnShape {
    uint32_t group, rows_log2, keys_log2, extra;
    uint32_t closed;                            // P is a whole number, and what it divides stays below 2^31
    AttnDivisor per;                            // P
};
// most_keys: no sequence has more
ATLAS_HD inline AttnShape attn_shape(uint32_t group, uint32_t rows_log2, uint32_t keys_log2, uint32_t extra, uint64_t most_keys, uint64_t most_rows) {
    const uint64_t k = uint64_t(group) << keys_log2, p = k >> rows_log2;
    const bool closed = (p << rows_log2) == k && p > 0 && p < (1ull << 31) && ((((most_keys + (1ull << keys_log2)) * group + most_rows) >> rows_log2) + 2) < (1ull << 31);
    return AttnShape{group, rows_log2, keys_log2, extra, closed ? 1u : 0u, attn_divisor(closed ? uint32_t(p) : 1u)};
}

// One sequence's blocks.  Without new tokens it has none; with fewer cached tokens than new ones (the first rows see nothing) all of
// its blocks count as if they saw the whole cache.
struct AttnSeq {
    uint32_t q_len, kv_len, blocks, whole;      // whole: tiles of the cached tokens, one at least
    uint32_t first;                             // floor(c / R)
    AttnShape sh;
    ATLAS_HD AttnSeq(uint32_t q, uint32_t kv, const AttnShape& shape) : q_len(q), kv_len(kv), sh(shape) {
        const uint32_t rows = 1u << sh.rows_log2;
        blocks = uint32_t((uint64_t(q) * sh.group + rows - 1) >> sh.rows_log2);
        whole = kv ? ((kv - 1) >> sh.keys_log2) + 1 : 1;
        first = uint32_t(numerator() >> sh.rows_log2);
    }
    // of block 0: its last row is row R - 1, token floor of that / group; it sees kv_len - q_len + that token + 1 keys
    ATLAS_HD uint64_t numerator() const { return ((1u << sh.rows_log2) - 1u) + uint64_t(sh.group) * (uint64_t(kv_len - q_len) + (1u << sh.keys_log2)); }
    ATLAS_HD uint32_t tiles(uint32_t b) const {
        if (kv_len < q_len || b + 1 >= blocks) return whole;
        const uint64_t t = sh.closed ? attn_div(first + b, sh.per) : attn_quotient((uint64_t(b) << sh.rows_log2) + numerator(), uint64_t(sh.group) << sh.keys_log2);
        return t < whole ? uint32_t(t) : whole;
    }
    // sum of floor(i / P) over i = 0 .. x - 1
    ATLAS_HD uint64_t upto(uint32_t x) const {
        const uint64_t q = attn_div(x, sh.per);
        return sh.per.d * (q * (q - 1) / 2) + q * (x - q * sh.per.d);
    }
    // places of the blocks before b, of one KV head
    ATLAS_HD uint64_t before(uint32_t b) const {
        if (b == 0 || blocks == 0) return 0;
        const uint32_t n = b < blocks ? b : blocks - 1;                                   // by the formula
        const uint64_t sum = n == 0 ? 0 : kv_len < q_len ? uint64_t(whole) * n : sh.closed ? upto(first + n) - upto(first)
                                      : floor_sum(n, uint64_t(sh.group) << sh.keys_log2, 1u << sh.rows_log2, numerator());
        return (b < blocks ? sum : sum + whole) + uint64_t(b) * sh.extra;
    }
    ATLAS_HD uint64_t total(uint32_t kv_heads) const { return before(blocks) * kv_heads; }
};

struct AttnPlace {
    uint32_t block, head, place, tiles;         // place within the item, which has extra + tiles of them
};
// where place x of a sequence's part of the line lies, known to be in a block
ATLAS_HD inline AttnPlace attn_place_in_block(const AttnSeq& s, uint32_t kv_heads, uint64_t x, uint32_t block) {
    AttnPlace p;
    p.block = block;
    p.tiles = s.tiles(block);
    const uint64_t in_block = x - s.before(block) * kv_heads;
    p.head = kv_heads == 1 ? 0u : uint32_t(attn_quotient(in_block, s.sh.extra + p.tiles));
    p.place = uint32_t(in_block - uint64_t(p.head) * (s.sh.extra + p.tiles));
    return p;
}
// How many of 32 candidates something holds for, looked at one after the other; a warp looks at them at once.
struct AttnOneByOne {
    template <typename F> ATLAS_HD uint32_t operator()(F holds) const {
        uint32_t n = 0;
        for (uint32_t i = 0; i < 32; ++i) n += holds(i) ? 1u : 0u;
        return n;
    }
};
// where place x of a sequence's part of the line lies, x < total(kv_heads)
template <typename Count = AttnOneByOne>
ATLAS_HD inline AttnPlace attn_locate(const AttnSeq& s, uint32_t kv_heads, uint64_t x, Count count = Count()) {
    uint32_t lo = 0, hi = s.blocks - 1;
    while (lo < hi) {                                                                     // the last block that begins at or before x
        const uint32_t step = (hi - lo + 31u) / 32u;
        const uint32_t past = count([&](uint32_t i) {
            const uint32_t mid = lo + (i + 1u) * step;
            return mid <= hi && s.before(mid) * kv_heads <= x;
        });
        lo += past * step;
        hi = hi < lo + step - 1u ? hi : lo + step - 1u;
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

// A line of `total` places, cut into as many ranges as there are CTAs, or fewer where each is to have `least` places at least.  The
// first `more` are one place longer.
struct AttnRanges {
    uint64_t total, each, more;
    uint32_t n;
    ATLAS_HD AttnRanges(uint64_t places, uint32_t ctas, uint32_t least) : total(places) {
        n = total >= uint64_t(ctas) * least ? ctas : total <= least ? 1u : uint32_t(attn_quotient(total + least - 1, least));
        each = attn_quotient(total, n);
        more = total - each * n;
    }
    ATLAS_HD uint64_t begin(uint32_t c) const { return each * c + (c < more ? c : more); }
    // the range that place x belongs to
    ATLAS_HD uint32_t of(uint64_t x) const {
        const uint64_t longer = more * (each + 1);
        return x < longer ? uint32_t(attn_quotient(x, each + 1)) : uint32_t(more + attn_quotient(x - longer, each));
    }
};

// How many pieces the item has that range c, beginning at `begin` and there at place `at`, cuts for the first time; 0 if it cuts none so.  A
// piece of an item is what a range has of its tiles: a cut among the places ahead of the first tile is none.
ATLAS_HD inline uint32_t attn_cut_pieces(const AttnRanges& r, uint32_t c, uint64_t begin, const AttnPlace& at, uint32_t extra) {
    const uint64_t first_tile = begin - at.place + extra;
    return c > 0 && begin > first_tile && r.begin(c - 1) <= first_tile ? r.of(first_tile + at.tiles - 1) - c + 2u : 0u;
}

}  // namespace atlas
