"""How the attention over the paged cache is cut into pieces (csrc/attn_plan.hpp), compiled for the host, against counting."""
import ctypes as C
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "apathy-atlas_b200", "csrc")

SOURCE = """
#include "attn_plan.hpp"
using namespace atlas;
extern "C" {
uint64_t floor_sum_(uint64_t n, uint64_t m, uint64_t a, uint64_t b) { return floor_sum(n, m, a, b); }
static AttnSeq seq_of(uint32_t q, uint32_t kv, uint32_t g, uint32_t r, uint32_t k, uint32_t e, uint64_t most) {
    uint32_t rl = 0, kl = 0;
    while ((1u << rl) < r) ++rl;
    while ((1u << kl) < k) ++kl;
    return AttnSeq(q, kv, attn_shape(g, rl, kl, e, most, uint64_t(q) * g));
}
uint32_t closed(uint32_t g, uint32_t r, uint32_t k, uint64_t most) { return seq_of(1, 1, g, r, k, 0, most).sh.closed; }
uint32_t tiles(uint32_t q, uint32_t kv, uint32_t g, uint32_t r, uint32_t k, uint32_t e, uint64_t most, uint32_t b) { return seq_of(q, kv, g, r, k, e, most).tiles(b); }
uint32_t blocks(uint32_t q, uint32_t kv, uint32_t g, uint32_t r, uint32_t k, uint32_t e, uint64_t most) { return seq_of(q, kv, g, r, k, e, most).blocks; }
uint64_t total(uint32_t q, uint32_t kv, uint32_t g, uint32_t r, uint32_t k, uint32_t e, uint64_t most, uint32_t h) { return seq_of(q, kv, g, r, k, e, most).total(h); }
int locate(uint32_t q, uint32_t kv, uint32_t g, uint32_t r, uint32_t k, uint32_t e, uint64_t most, uint32_t h, uint64_t x, uint32_t* out) {
    const AttnSeq s = seq_of(q, kv, g, r, k, e, most);
    AttnPlace p = attn_locate(s, h, x);
    out[0] = p.block; out[1] = p.head; out[2] = p.place; out[3] = p.tiles;
    const int more = attn_next(s, h, p);
    out[4] = p.block; out[5] = p.head; out[6] = p.place; out[7] = p.tiles;
    return more;
}
uint32_t divided(uint32_t x, uint32_t d) { return attn_div(x, attn_divisor(d)); }
uint64_t range_begin(uint64_t t, uint32_t ctas, uint32_t least, uint32_t c) { return AttnRanges(t, ctas, least).begin(c); }
uint32_t range_of(uint64_t t, uint32_t ctas, uint32_t least, uint64_t x) { return AttnRanges(t, ctas, least).of(x); }
uint32_t ranges(uint64_t t, uint32_t ctas, uint32_t least) { return AttnRanges(t, ctas, least).n; }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", "-o", str(d / "plan.so"), str(d / "plan.cpp")],
                   check=True)
    L = C.CDLL(str(d / "plan.so"))
    u32, u64 = C.c_uint32, C.c_uint64
    L.floor_sum_.argtypes, L.floor_sum_.restype = [u64] * 4, u64
    L.tiles.argtypes = [u32] * 6 + [u64, u32]
    L.blocks.argtypes = [u32] * 6 + [u64]
    L.closed.argtypes = [u32] * 3 + [u64]
    L.total.argtypes, L.total.restype = [u32] * 6 + [u64, u32], u64
    L.locate.argtypes = [u32] * 6 + [u64, u32, u64, C.POINTER(u32)]
    L.divided.argtypes, L.divided.restype = [u32, u32], u32
    L.range_begin.argtypes, L.range_begin.restype = [u64, u32, u32, u32], u64
    L.range_of.argtypes, L.range_of.restype = [u64, u32, u32, u64], u32
    L.ranges.argtypes, L.ranges.restype = [u64, u32, u32], u32
    return L


def test_floor_sum(plan):
    rng = random.Random(1)
    for _ in range(300):
        n, m, a, b = rng.randint(0, 60), rng.randint(1, 40), rng.randint(0, 90), rng.randint(0, 500)
        assert plan.floor_sum_(n, m, a, b) == sum((a * i + b) // m for i in range(n))


def _counted(q, kv, g, rows, keys):
    """Tiles of every block of rows, by looking at what its last row sees."""
    n = -(-q * g // rows)
    out = []
    for b in range(n):
        last = min(q - 1, ((b + 1) * rows - 1) // g)
        seen = kv if kv < q else kv - q + last + 1
        out.append(max(1, -(-seen // keys)))
    return out


def test_divisors(plan):
    rng = random.Random(2)
    for d in [1, 2, 3, 5, 7, 16, 24, 100, 4095, 65537, (1 << 30) + 1, (1 << 31) - 1] + [rng.randint(1, 1 << 31) for _ in range(50)]:
        for x in [0, 1, d - 1, d, d + 1, 2 * d - 1, (1 << 31) - 1] + [rng.randint(0, (1 << 31) - 1) for _ in range(20)]:
            if x < 1 << 31:
                assert plan.divided(x, d) == x // d


@pytest.mark.parametrize("most", [5000, 1 << 30], ids=["closed", "by_floor_sum"])
@pytest.mark.parametrize("rows,keys,extra", [(8, 64, 1), (16, 64, 1), (16, 128, 0), (128, 128, 2), (256, 128, 3)])
def test_blocks_and_places(plan, rows, keys, extra, most):
    rng = random.Random(rows + keys)
    out = (C.c_uint32 * 8)()
    assert plan.closed(4, rows, keys, 5000) == 1 and plan.closed(3, 256, 128, 5000) == 0 and plan.closed(64, rows, keys, 1 << 30) == (rows > 32)
    for _ in range(150):
        g, h = rng.choice((1, 2, 3, 4, 5, 7, 8, 16, 40)), rng.choice((1, 2, 5))
        q = rng.choice((1, 1, 2, rng.randint(1, 40), rng.randint(1, 700)))
        kv = rng.choice((q, q + rng.randint(0, 400), rng.randint(0, q), q + 64, q + 127))
        tiles, how = _counted(q, kv, g, rows, keys), (q, kv, g, rows, keys, extra, most)
        assert plan.blocks(*how) == len(tiles)
        assert [plan.tiles(*how, b) for b in range(len(tiles))] == tiles
        assert plan.total(*how, h) == h * (sum(tiles) + extra * len(tiles))
        x, items = 0, [(b, head, t) for b, t in enumerate(tiles) for head in range(h)]
        for i, (b, head, t) in enumerate(items):
            for place in {0, (t + extra) // 2, t + extra - 1}:
                more = plan.locate(*how, h, x + place, out)
                assert tuple(out)[:4] == (b, head, place, t)
                assert bool(more) == (i + 1 < len(items))
                if more:
                    assert tuple(out)[4:] == (items[i + 1][0], items[i + 1][1], 0, items[i + 1][2])
            x += t + extra
    assert plan.blocks(0, 77, 4, rows, keys, extra, most) == 0 and plan.total(0, 77, 4, rows, keys, extra, most, 8) == 0


def test_ranges_cover_the_line(plan):
    rng = random.Random(3)
    for _ in range(100):
        total, ctas, least = rng.randint(1, 3000), rng.randint(1, 400), rng.randint(1, 9)
        n = plan.ranges(total, ctas, least)
        assert 1 <= n <= ctas and (n == 1 or (n - 1) * least < total)
        begins = [plan.range_begin(total, ctas, least, c) for c in range(n + 1)]
        assert begins[0] == 0 and begins[-1] == total
        sizes = [b - a for a, b in zip(begins, begins[1:])]
        assert max(sizes) - min(sizes) <= 1 and min(sizes) >= 1
        for c in range(n):
            assert plan.range_of(total, ctas, least, begins[c]) == c and plan.range_of(total, ctas, least, begins[c + 1] - 1) == c
    assert plan.ranges(0, 148, 4) == 1
    assert plan.range_begin(1 << 45, 148, 1, 147) == (1 << 45) // 148 * 147 + min(147, (1 << 45) % 148)
