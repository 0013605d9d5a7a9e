"""Where the ranges of the attention's line of tiles cut items, and into how many pieces (csrc/attn_plan.hpp), compiled for the host, against counting."""
import ctypes as C
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "apathy-atlas_b200", "csrc")

SOURCE = """
#include "attn_plan.hpp"
using namespace atlas;
// Of every range of a line of sequences: where it begins (sequence, block, head, place, tiles) and the pieces that it notes.
extern "C" uint32_t notes(uint32_t n_seqs, const uint32_t* q, const uint32_t* kv, uint32_t group, uint32_t rows_log2, uint32_t keys_log2, uint32_t extra, uint32_t heads,
                          uint32_t ctas, uint32_t least, uint32_t* out) {
    uint64_t most_rows = 0, most_keys = 0, total = 0;
    for (uint32_t s = 0; s < n_seqs; ++s) { most_rows += uint64_t(q[s]) * group; most_keys = kv[s] > most_keys ? kv[s] : most_keys; }
    const AttnShape shape = attn_shape(group, rows_log2, keys_log2, extra, most_keys, most_rows);
    for (uint32_t s = 0; s < n_seqs; ++s) total += AttnSeq(q[s], kv[s], shape).total(heads);
    const AttnRanges r(total, ctas, least);
    for (uint32_t c = 0; c < r.n; ++c) {
        const uint64_t begin = r.begin(c);
        uint64_t before = 0;
        for (uint32_t s = 0; s < n_seqs; ++s) {
            const AttnSeq plan(q[s], kv[s], shape);
            const uint64_t places = plan.total(heads);
            if (begin < before + places) {
                const AttnPlace at = attn_locate(plan, heads, begin - before);
                uint32_t* o = out + 6 * c;
                o[0] = s; o[1] = at.block; o[2] = at.head; o[3] = at.place; o[4] = at.tiles;
                o[5] = attn_cut_pieces(r, c, begin, at, extra);
                break;
            }
            before += places;
        }
    }
    return r.n;
}
"""


@pytest.fixture(scope="module")
def notes(tmp_path_factory):
    d = tmp_path_factory.mktemp("cuts")
    (d / "cuts.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", "-o", str(d / "cuts.so"), str(d / "cuts.cpp")], check=True)
    f = C.CDLL(str(d / "cuts.so")).notes
    u32 = C.c_uint32
    f.argtypes, f.restype = [u32, C.POINTER(u32), C.POINTER(u32)] + [u32] * 7 + [C.POINTER(u32)], u32
    return f


@pytest.mark.parametrize("rows_log2,keys_log2,extra", [(3, 6, 2), (4, 7, 2), (4, 6, 0), (7, 7, 1), (8, 7, 2)])
def test_cuts_against_counting(notes, rows_log2, keys_log2, extra):
    rng = random.Random(rows_log2 * 100 + keys_log2 * 10 + extra)
    rows, keys = 1 << rows_log2, 1 << keys_log2
    for _ in range(120):
        group, heads = rng.choice((1, 2, 3, 4, 5, 8)), rng.choice((1, 2, 4))
        ctas, least = rng.choice((1, 2, 7, 148, 444)), rng.choice((1, 2, 4))
        lens = []
        for _ in range(rng.randint(1, 6)):
            q = rng.choice((0, 1, 1, 2, rng.randint(1, 300), rng.randint(1, 3000)))
            lens.append((q, q + rng.choice((0, 1, rng.randint(0, 500), rng.randint(0, 20000))) if rng.random() < 0.9 else rng.randint(0, q)))
        line = []                                              # (sequence, block, head, tiles), in the order of the line
        for s, (q, kv) in enumerate(lens):
            blocks = -(-q * group // rows)
            for b in range(blocks):
                last = min(q - 1, ((b + 1) * rows - 1) // group)
                seen = kv if kv < q else kv - q + last + 1
                line += [(s, b, h, max(1, -(-seen // keys))) for h in range(heads)]
        if not line:
            continue
        q_arr, kv_arr = ((C.c_uint32 * len(lens))(*(x[i] for x in lens)) for i in range(2))
        out = (C.c_uint32 * (6 * ctas))()
        n = notes(len(lens), q_arr, kv_arr, group, rows_log2, keys_log2, extra, heads, ctas, least, out)
        total = sum(t + extra for *_, t in line)
        size, more = divmod(total, n)
        begins = [c * size + min(c, more) for c in range(n + 1)]
        pieces_of, at = {}, 0                                  # the first range that begins behind an item's first tile -> its pieces
        where = {}
        for s, b, h, t in line:
            first, end = at + extra, at + extra + t
            holders = [c for c in range(n) if begins[c] < end and begins[c + 1] > first]
            if len(holders) > 1:
                assert holders == list(range(holders[0], holders[-1] + 1))
                pieces_of[holders[1]] = len(holders)
            for c in range(n):
                if at <= begins[c] < end:
                    where[c] = (s, b, h, begins[c] - at, t)
            at = end
        for c in range(n):
            assert tuple(out[6 * c:6 * c + 5]) == where[c], c
            assert out[6 * c + 5] == pieces_of.get(c, 0), c
