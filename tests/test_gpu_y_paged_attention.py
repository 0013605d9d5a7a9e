"""Attention over the paged K/V cache against the same in 64 bits, with bounds derived from its arithmetic (attention_util.Batch.exact):
one new token to many, odd lengths, pages that end inside a tile, both cache types, all head sizes, rows that see nothing, stale NaN
behind every sequence, padded batches, cuts of long sequences."""
import math

import pytest

from attention_util import Batch

pytestmark = pytest.mark.gpu

DECODE = [
    # lens, heads, kv_heads, d, page
    ([(1, 1)], 1, 1, 64, 16),
    ([(1, 777)], 32, 8, 128, 16),
    ([(1, 63), (1, 64), (1, 65), (1, 1), (1, 200)], 8, 2, 128, 16),
    ([(1, 5000), (1, 17), (0, 44), (1, 129)], 16, 2, 128, 24),
    ([(1, 9000), (1, 9001)], 8, 1, 64, 5),
    ([(1, 300), (1, 4097)], 7, 1, 96, 1),
    ([(1, 1023), (1, 1)], 16, 1, 256, 256),
    ([(1, 450)] * 40, 4, 4, 128, 64),
    ([(1, 333), (1, 2)], 3, 3, 32, 7),
    ([(1, 515)], 24, 1, 160, 16),
    ([(1, 40000)], 4, 1, 128, 128),
]
CHUNK = [
    ([(5, 5), (3, 700), (7, 64), (1, 128)], 8, 2, 128, 16),
    ([(16, 1000), (2, 2)], 64, 8, 128, 32),
    ([(33, 33), (0, 10), (40, 333)], 6, 2, 64, 24),
    ([(130, 257), (1, 1)], 4, 1, 256, 16),
    ([(77, 901)], 12, 4, 96, 13),
    ([(200, 200), (129, 2000)], 8, 8, 128, 16),
    ([(9, 4), (3, 0), (6, 6)], 4, 2, 128, 16),          # rows that see nothing; a sequence without any key
    ([(513, 3001)], 7, 1, 128, 64),
    ([(64, 64), (65, 65), (63, 63), (127, 127), (128, 128)], 2, 1, 64, 8),
]


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("case", DECODE + CHUNK, ids=lambda c: f"{c[0][0][0]}x{c[0][0][1]}_{c[1]}_{c[2]}_{c[3]}_{c[4]}")
def test_against_64_bits(cuda, atlas, case, fp8):
    lens, heads, kv_heads, d, page = case
    b = Batch(cuda, atlas, lens, heads, kv_heads, d, page, fp8, seed=d + page)
    atlas.paged_attention(b.desc())
    b.check()


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
def test_without_scratch_and_without_lse(cuda, atlas, fp8):
    b = Batch(cuda, atlas, [(1, 3000), (4, 900), (1, 20)], 8, 2, 128, 16, fp8, seed=3)
    atlas.paged_attention(b.desc(ws=False, lse=False))
    b.check(lse=False)
    assert atlas.last_attention_shape()["whole_items"]


def test_strided_q_and_out(cuda, atlas):
    b = Batch(cuda, atlas, [(1, 500), (3, 77), (130, 400)], 8, 2, 128, 16, seed=4, q_extra=264)
    wide = cuda.full((b.rows + 3, b.heads * b.d + 40), 77.0, dtype=cuda.bfloat16, device="cuda")
    atlas.paged_attention(b.desc(out=wide, out_row_stride=wide.shape[1]))
    assert (wide[:, b.heads * b.d:] == 77.0).all()
    b.out = wide[:, :b.heads * b.d].contiguous()
    b.check()


@pytest.mark.parametrize("lens", [[(1, 20000), (1, 31)], [(300, 2500), (40, 41)]], ids=["decode", "chunk"])
def test_same_call_same_bits(cuda, atlas, lens):
    b = Batch(cuda, atlas, lens, 8, 2, 128, 16, seed=5)
    d = b.desc()
    atlas.paged_attention(d)
    cuda.cuda.synchronize()
    first = b.out.clone(), b.lse.clone()
    for _ in range(3):
        b.out.fill_(1.0)
        b.ws.fill_(math.nan)
        atlas.paged_attention(d)
    cuda.cuda.synchronize()
    assert cuda.equal(b.out[:b.rows], first[0][:b.rows]) and cuda.equal(b.lse, first[1])


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 8), (256, 16), (128, 5)])
def test_values_of_later_tokens_stay_theirs(cuda, atlas, fp8, d, page):
    """Infinite and NaN values of a token reach the rows that see it and no others."""
    torch = cuda
    b = Batch(cuda, atlas, [(40, 333), (300, 301), (4, 4)], 8, 2, d, page, fp8, seed=6)
    slots = b.slots(1, 301)
    bad = [200, 290]
    if fp8:
        b.v.view(torch.uint8)[slots[bad[0]], 1, 3] = 0x7F
        b.v.view(torch.uint8)[slots[bad[1]], 0, :] = 0xFF
    else:
        b.v[slots[bad[0]], 1, 3] = math.nan
        b.v[slots[bad[1]], 0, :] = math.inf
    desc = b.desc()
    atlas.paged_attention(desc)
    torch.cuda.synchronize()
    got = b.out[:b.rows].float().view(b.rows, 2, 4, d)
    for h, first, cols in ((1, bad[0], [3]), (0, bad[1], list(range(d)))):
        seen = torch.zeros((300, d), dtype=torch.bool, device="cuda")
        seen[first - 1:, cols] = True                              # new token i stands at position i + 1
        odd = ~torch.isfinite(got[40:340, h])
        assert torch.equal(odd, seen[:, None].expand(-1, 4, -1))
    assert torch.isfinite(got[:40]).all() and torch.isfinite(got[340:]).all()
    # rows that do not see them are what they are without them
    keep = got.clone()
    if fp8:
        b.v.view(torch.uint8)[torch.from_numpy(slots[bad]).cuda()] = 0
    else:
        b.v[torch.from_numpy(slots[bad]).cuda()] = 0
    atlas.paged_attention(desc)
    torch.cuda.synchronize()
    clean = b.out[:b.rows].float().view(b.rows, 2, 4, d)
    fine = torch.isfinite(keep)
    rows = torch.arange(b.rows, device="cuda")
    unseen = (rows < 40 + bad[0] - 1) | (rows >= 340)
    tol = 2.0 ** -6 * (clean.abs() + 1.0)                          # (a row computed again adds in another order, P unrounded)
    assert ((keep - clean).abs() <= tol)[unseen].all() and fine[unseen].all()


def test_scores_with_infinities(cuda, atlas):
    """A key of infinite values: a NaN or infinite score makes its row NaN, as the formula has it, and no other row."""
    b = Batch(cuda, atlas, [(1, 100), (1, 100)], 4, 1, 64, 16, seed=7)
    b.k[b.slots(0, 100)[50]] = math.inf
    atlas.paged_attention(b.desc())
    cuda.cuda.synchronize()
    assert cuda.isnan(b.out[0].float()).all() and cuda.isfinite(b.out[1].float()).all()


def test_pages_that_do_not_exist_read_as_zeros(cuda, atlas):
    b = Batch(cuda, atlas, [(1, 200), (1, 90)], 8, 2, 128, 16, seed=8)
    for bad in (-1, b.n_pages, 0x7FFFFFFF):
        b.table[0, 3] = bad
        atlas.paged_attention(b.desc())
        cuda.cuda.synchronize()
        assert atlas.device_status() == 4
        k, v = b.k, b.v
        slots = b.slots(0, 200)
        out = b.out[0].double().view(8, 128)
        for h in range(8):
            kk, vv = k[slots, h // 4].double(), v[slots, h // 4].double()
            kk[48:64] = 0
            vv[48:64] = 0
            p = cuda.softmax(kk @ b.q[0, h * 128:(h + 1) * 128].double() * b.scale, 0)
            assert (p @ vv - out[h]).abs().max() <= 2.0 ** -6 * (p @ vv.abs()).max()
    # a length beyond the table's row: what fits is taken
    b.table[0, 3] = int(b.table_np[0, 3])
    b.table[1, :] = b.table[0, :]
    b.table[:, -1] = b.table[:, 0]
    b.kv[0] = b.kv[1] = 0x7FFFFFFF
    atlas.paged_attention(b.desc())
    cuda.cuda.synchronize()
    assert atlas.device_status() == 5


def test_captured_with_other_lengths(cuda, atlas):
    """A captured call follows the lengths and tables that stand there when it is replayed, padded batches among them."""
    torch = cuda
    b = Batch(cuda, atlas, [(1, 3000), (1, 500), (1, 64), (1, 1)], 8, 2, 128, 16, seed=9)
    d = b.desc()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        atlas.paged_attention(d)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            atlas.paged_attention(d)
    for lens in ([(1, 2999), (1, 3), (1, 60), (1, 1)], [(1, 1), (1, 499), (0, 0), (0, 0)], [(1, 3000), (1, 500), (1, 64), (1, 1)]):
        b.lens = lens
        b.cu_np[1:] = [sum(q for q, _ in lens[:i + 1]) for i in range(4)]
        b.cu.copy_(torch.from_numpy(b.cu_np))
        b.kv.copy_(torch.tensor([kv for _, kv in lens], dtype=torch.int32))
        b.rows = int(b.cu_np[-1])
        b.out.fill_(77.0)
        b.lse.fill_(77.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        b.check()


def test_two_streams(cuda, atlas):
    torch = cuda
    batches = [Batch(cuda, atlas, [(1, 30000), (1, 100 * i + 1)], 8, 2, 128, 16, seed=10 + i) for i in range(2)]
    descs, streams = [b.desc() for b in batches], [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    for _ in range(20):
        for d, s in zip(descs, streams):
            atlas.paged_attention(d, stream=s)
    torch.cuda.synchronize()
    for b in batches:
        b.check()


def test_large_pool_beyond_32_bits(cuda, atlas):
    """Byte offsets into the cache pass 2^32: pages at the pool's far end."""
    torch = cuda
    pages, page, hk, d = 40000, 32, 8, 128                          # 2.6 GB a side, 1.3 G values
    k, v = (torch.zeros((pages * page, hk, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    b = Batch(cuda, atlas, [(1, 300), (70, 300)], 16, 8, d, page, seed=12)
    far = pages - b.n_pages
    k[far * page:].copy_(b.k)
    v[far * page:].copy_(b.v)
    b.table += far
    atlas.paged_attention(b.desc(k_cache=k, v_cache=v, n_pages=pages))
    b.check()
