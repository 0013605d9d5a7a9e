"""Paged attention at the edges of what its description allows: more sequences than one warp sums up, clusters that share an item, lengths
beyond the promised ones, tables that are wrong, which kernel a call takes, values that are not finite in a long cache."""
import ctypes
import math

import numpy as np
import pytest

from attention_util import Batch

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])


@BOTH
@pytest.mark.parametrize("n,chunk", [(257, 1), (1500, 1), (300, 5), (600, 40)])
def test_many_sequences(cuda, atlas, n, chunk, fp8):
    """Beyond 256 sequences all warps of a CTA sum up the line of tiles; empty sequences and sequences without new tokens among them."""
    rng = np.random.default_rng(n)
    lens = [(int(q), int(q) + int(k)) for q, k in zip(rng.integers(0, chunk + 1, n), rng.integers(0, 90, n))]
    lens[n // 2] = (chunk, 3000)
    b = Batch(cuda, atlas, lens, 4, 2, 64, 16, fp8, seed=n)
    atlas.paged_attention(b.desc())
    b.check()


@BOTH
@pytest.mark.parametrize("lens,heads,kv_heads,d", [
    ([(1, 777)], 32, 8, 128), ([(1, 129)], 1, 1, 128), ([(1, 1000 - 111 * i) for i in range(8)], 32, 8, 128), ([(2, 600), (1, 5), (2, 2)], 8, 2, 64),
    ([(1, 500), (0, 300), (1, 1), (1, 0)], 6, 2, 256), ([(4, 700), (3, 70)], 12, 4, 96), ([(1, 1024)] * 4, 4, 4, 32)])
def test_clusters(cuda, atlas, lens, heads, kv_heads, d, fp8):
    b = Batch(cuda, atlas, lens, heads, kv_heads, d, 16, fp8, seed=d)
    desc = b.desc()
    atlas.paged_attention(desc)
    b.check()
    shape, items = atlas.last_attention_shape(), len(lens) * kv_heads
    assert shape["whole_items"] and shape["ctas"] in (2 * items, 4 * items, 8 * items)
    first = b.out.clone()
    b.out.fill_(77.0)
    atlas.paged_attention(desc)
    b.check()
    assert cuda.equal(b.out, first)


@BOTH
def test_clusters_over_a_long_cache_without_scratch(cuda, atlas, fp8):
    b = Batch(cuda, atlas, [(1, 20000), (1, 3)], 8, 2, 128, 16, fp8, seed=2)
    atlas.paged_attention(b.desc(ws=False))
    b.check()
    assert atlas.last_attention_shape()["ctas"] == 32


@BOTH
@pytest.mark.parametrize("lens,promise", [([(1, 5000), (1, 40)], (1, 60)), ([(1, 700)] * 3, (1, 1)), ([(30, 900), (2, 30)], (1, 200)),
                                          ([(130, 2600), (200, 200)], (20, 100)), ([(130, 2600), (200, 200)], (1, 100))])
def test_more_than_promised(cuda, atlas, lens, promise, fp8):
    """Longer sequences than max_q_len and max_kv_len are computed all the same."""
    b = Batch(cuda, atlas, lens, 8, 2, 128, 16, fp8, seed=3)
    atlas.paged_attention(b.desc(max_q_len=promise[0], max_kv_len=promise[1]))
    b.check()


@BOTH
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 256])
@pytest.mark.parametrize("page", [1, 5, 12])
def test_chunks_over_pages_of_any_size(cuda, atlas, page, d, fp8):
    """Pages that no box of eight rows divides: tiles of keys are gathered row by row."""
    b = Batch(cuda, atlas, [(70, 1111), (33, 33), (0, 9), (257, 300), (1, 128)], 4, 2, d, page, fp8, seed=d + page)
    atlas.paged_attention(b.desc())
    assert atlas.last_attention_shape()["block_rows"] == (256 if d <= 128 else 128)
    b.check()


@BOTH
@pytest.mark.parametrize("heads,lens", [(3, [(700, 3000), (90, 700), (301, 301)]), (5, [(257, 900), (1, 4), (600, 601)]), (7, [(110, 4000), (37, 38)])])
def test_blocks_that_begin_inside_a_token(cuda, atlas, heads, lens, fp8):
    """Groups that do not divide a block: a token's heads lie in two blocks, and the line of tiles has no period."""
    b = Batch(cuda, atlas, lens, heads, 1, 128, 16, fp8, seed=heads)
    atlas.paged_attention(b.desc())
    b.check()


def test_which_kernel(cuda, atlas):
    def rows(lens, heads, kv_heads, d=128, page=16, fp8=False, q_extra=0, **kw):
        b = Batch(cuda, atlas, lens, heads, kv_heads, d, page, fp8, seed=4, q_extra=q_extra)
        atlas.paged_attention(b.desc(**kw))
        b.check()
        return atlas.last_attention_shape()["block_rows"]

    assert rows([(1, 300)], 8, 1) == 8 and rows([(1, 300)], 9, 1) == 16 and rows([(2, 300)], 8, 1) == 16
    assert rows([(1, 300)], 17, 1) == 256 and rows([(3, 300)], 8, 1, d=256) == 128
    assert rows([(4, 300)], 8, 1, fp8=True) == 16 and rows([(5, 300)], 8, 1, fp8=True) == 256
    assert rows([(9, 300)], 8, 1, page=4) == 256                   # pages that no box of eight rows fits: row by row
    assert rows([(9, 300)], 8, 1, page=24) == 256                  # boxes of eight
    assert rows([(9, 300)], 8, 1, q_extra=2) == 16                 # rows of q that are not on 16 bytes


@BOTH
def test_q_and_out_at_odd_addresses(cuda, atlas, fp8):
    torch = cuda
    b = Batch(cuda, atlas, [(33, 500), (1, 77)], 8, 2, 128, 16, fp8, seed=5)
    flat = torch.zeros(b.q.numel() + 2, dtype=torch.bfloat16, device="cuda")
    q = flat[2:].view(b.q.shape)
    q.copy_(b.q)
    wide = torch.full((b.rows + 3, b.heads * b.d + 1), 77.0, dtype=torch.bfloat16, device="cuda")
    out = wide.flatten()[1:]                                       # 2-byte aligned, rows an odd number of elements apart
    atlas.paged_attention(b.desc(q=q, out=out, out_row_stride=wide.shape[1]))
    torch.cuda.synchronize()
    b.out[:b.rows] = wide[:b.rows, 1:]
    assert (wide[1:b.rows, 0] == 77.0).all()
    b.check()


@BOTH
@pytest.mark.parametrize("page", [16, 4])
def test_wrong_tables_under_a_chunk(cuda, atlas, page, fp8):
    """A page that is not of the pool reads as zeros; a length beyond the table's row is cut to it."""
    b = Batch(cuda, atlas, [(40, 333), (20, 90)], 8, 2, 128, page, fp8, seed=6)
    for bad in (-1, b.n_pages, 0x7FFFFFFF):
        keep = int(b.table_np[0, 3])
        b.table[0, 3] = bad
        atlas.paged_attention(b.desc())
        cuda.cuda.synchronize()
        assert atlas.last_attention_shape()["block_rows"] == 256 and atlas.device_status() == 4
        got, got_l = b.out.clone(), b.lse.clone()
        b.table[0, 3] = keep
        at = cuda.from_numpy(b.slots(0, 333)[3 * page:4 * page]).cuda()
        sides = [t.view(cuda.uint8) for t in (b.k, b.v)]
        held = [t[at].clone() for t in sides]
        for t in sides:
            t[at] = 0
        b.out.copy_(got)
        b.lse.copy_(got_l)
        b.check()
        for t, was in zip(sides, held):
            t[at] = was
    b.table[0, :] = b.table[0, 0]
    b.kv[0] = 0x7FFFFFFF
    atlas.paged_attention(b.desc())
    cuda.cuda.synchronize()
    assert atlas.device_status() == 5 and cuda.isfinite(b.out[:b.rows].float()).all()


@BOTH
@pytest.mark.parametrize("heads", [4, 40])
def test_rows_and_lengths_that_cannot_be(cuda, atlas, heads, fp8):
    """Ends of rows below zero, behind the buffer or ahead of their beginning; lengths below zero."""
    b = Batch(cuda, atlas, [(3, 50), (0, 40), (5, 60)], heads, 2, 64, 16, fp8, seed=7)
    desc = b.desc()
    b.cu.copy_(cuda.tensor([-9, 3, 3, 0x7FFFFFFF], dtype=cuda.int32))         # 0 .. 2, none, 3 .. 7
    atlas.paged_attention(desc)
    b.check()
    b.cu.copy_(cuda.tensor([8, 3, -7, -8], dtype=cuda.int32))                 # no rows at all
    b.out.fill_(77.0)
    b.lse.fill_(77.0)
    atlas.paged_attention(desc)
    cuda.cuda.synchronize()
    assert (b.out == 77.0).all() and (b.lse == 77.0).all()
    b.cu.copy_(cuda.from_numpy(b.cu_np))
    b.kv[2] = -5
    atlas.paged_attention(desc)
    cuda.cuda.synchronize()
    assert (b.out[3:8] == 0.0).all() and (b.lse[3:8] == -math.inf).all()
    assert atlas.device_status() == 0


@BOTH
def test_nothing_but_empty_sequences(cuda, atlas, fp8):
    b = Batch(cuda, atlas, [(1, 0), (1, 0)], 8, 2, 128, 16, fp8, seed=8)
    atlas.paged_attention(b.desc())
    b.check()


@BOTH
@pytest.mark.parametrize("side", ["k", "v"])
def test_not_finite_in_a_long_cache(cuda, atlas, side, fp8):
    """What every row sees stays in its channel (its head, if it is a key's) and takes no time worth mentioning; what only the last rows
    see reaches none before them, however many keys these have."""
    torch = cuda
    n, new, d = 60000, 40, 128
    b = Batch(cuda, atlas, [(new, n), (3, 9)], 16, 2, d, 16, fp8, seed=9)
    cache = b.v if side == "v" else b.k
    slots = b.slots(0, n)

    def plant(token, head, ch):
        if fp8:
            cache.view(torch.uint8)[slots[token], head, ch] = 0x7F
        else:
            cache[slots[token], head, ch] = math.nan

    plant(0, 0, 5)
    plant(n - 10, 1, 7)
    desc = b.desc()
    t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    t0.record()
    atlas.paged_attention(desc)
    t1.record()
    torch.cuda.synchronize()
    assert atlas.device_status() == 0 and t0.elapsed_time(t1) < 500.0
    odd = ~torch.isfinite(b.out[:b.rows].float().view(b.rows, 2, 8, d))
    want = torch.zeros_like(odd)
    want[:new, 0, :, 5 if side == "v" else slice(None)] = True
    want[new - 10:new, 1, :, 7 if side == "v" else slice(None)] = True
    assert torch.equal(odd, want)
    for t in (0, n - 10):
        cache.view(torch.uint8)[slots[t]] = 0
    got = b.out[:b.rows].clone()
    atlas.paged_attention(desc)
    torch.cuda.synchronize()
    b.check()
    if side == "v":
        # the rows ahead of the second one have all but that token's share, which was not theirs to see
        same = ~want
        same[:, 0] = False                                         # (token 0's other channels have changed)
        same[new - 10:new] = False
        a, c = got.double().view(same.shape)[same], b.out[:b.rows].double().view(same.shape)[same]
        assert ((a - c).abs() <= 2.0 ** -6 * (c.abs() + 1.0)).all()


def test_scratch(cuda, atlas):
    """Too little of it, or not where it may be: refused before anything runs."""
    b = Batch(cuda, atlas, [(1, 9000)], 8, 2, 128, 16, seed=10)
    d = b.desc()
    assert d.ws_bytes > 0
    d.ws_bytes -= 4
    assert atlas.lib().atlas_b200_paged_attention(ctypes.byref(d), None) == -2
    d.ws_bytes += 4
    d.ws += 16
    assert atlas.lib().atlas_b200_paged_attention(ctypes.byref(d), None) == -3
    cuda.cuda.synchronize()
    assert (b.out == 77.0).all()


@BOTH
def test_captured_chunks(cuda, atlas, fp8):
    """Two captured calls of chunks, on scratch of their own, follow what stands in lengths, rows and tables when they are replayed."""
    torch = cuda
    batches = [Batch(cuda, atlas, [(100, 2000), (60, 500), (9, 64)], 8, 2, 128, 16, fp8, seed=11 + i) for i in range(2)]
    descs, graphs, side = [b.desc() for b in batches], [torch.cuda.CUDAGraph() for _ in batches], torch.cuda.Stream()
    with torch.cuda.stream(side):
        for d, g in zip(descs, graphs):
            with torch.cuda.graph(g, stream=side):
                atlas.paged_attention(d)
    for lens in ([(100, 2000), (60, 500), (9, 64)], [(1, 1), (77, 499), (0, 0)], [(3, 2000), (1, 500), (9, 9)]):
        for b in batches:
            b.lens = lens
            b.cu_np[1:] = [sum(q for q, _ in lens[:i + 1]) for i in range(3)]
            b.cu.copy_(torch.from_numpy(b.cu_np))
            b.kv.copy_(torch.tensor([kv for _, kv in lens], dtype=torch.int32))
            b.rows = int(b.cu_np[-1])
            b.out.fill_(77.0)
            b.lse.fill_(77.0)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for b in batches:
            b.check()
