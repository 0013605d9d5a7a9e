"""The operators around the paged cache with byte offsets beyond 2^32: pages at the far end of pools of 4.9 GB a side, in every form."""
import numpy as np
import pytest

from attention_util import Batch

pytestmark = pytest.mark.gpu

BYTES = 4_900_000_000


@pytest.fixture(scope="module")
def sides(cuda):
    two = [cuda.zeros(BYTES, dtype=cuda.uint8, device="cuda") for _ in range(2)]
    yield two
    del two
    cuda.cuda.empty_cache()


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("lens,heads,page,block_rows", [([(1, 300), (1, 5000)], 8, 16, 8), ([(3, 300), (1, 40)], 32, 16, 16), ([(70, 300), (1, 2000)], 32, 16, 256),
                                                        ([(70, 300), (1, 2000)], 32, 5, 256), ([(1, 500)], 8, 1, 8)])
def test_attention(cuda, atlas, sides, lens, heads, page, block_rows, fp8):
    torch, kv_heads, d = cuda, 8, 128
    row = kv_heads * d * (1 if fp8 else 2)
    pages = BYTES // (row * page)
    b = Batch(cuda, atlas, lens, heads, kv_heads, d, page, fp8, seed=page)
    far = pages - b.n_pages
    assert far * page * row > 1 << 32 and pages * page < 1 << 31
    kind = torch.float8_e4m3fn if fp8 else torch.bfloat16
    k, v = (t[:pages * page * row].view(kind).view(-1, kv_heads, d) for t in sides)
    for t, own in ((k, b.k), (v, b.v)):
        t[far * page:] = own
    b.table[:] = torch.where(b.table < b.n_pages, b.table + far, b.table)
    atlas.paged_attention(b.desc(k_cache=k, v_cache=v, n_pages=pages))
    assert atlas.last_attention_shape()["block_rows"] == block_rows
    b.check()


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("d,rot", [(128, 64), (128, 128), (128, 32)])
def test_writer(cuda, atlas, sides, d, rot, fp8):
    """The same tokens into the pool's last rows and into a small cache: the same bytes."""
    torch, hq, hk, tokens = cuda, 4, 2, 5
    row = hk * d * (1 if fp8 else 2)
    g = torch.Generator(device="cuda")
    g.manual_seed(d + rot)
    width = (hq + 2 * hk) * d
    qkv = torch.randn((tokens, width), generator=g, device="cuda").to(torch.bfloat16)
    w = [(torch.randn(d, generator=g, device="cuda") * 0.2).to(torch.bfloat16) for _ in range(2)]
    pos = torch.arange(tokens, dtype=torch.int32, device="cuda") * 1000
    freq = (1e6 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)).float()
    n_rows = BYTES // row
    small = [torch.zeros(16 * row, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for caches, first in ((sides, n_rows - tokens), (small, 0)):
        buf, slots = qkv.clone(), torch.arange(tokens, device="cuda") + first
        p = buf.data_ptr()
        args = (p, p + 2 * hq * d, p + 2 * (hq + hk) * d, width, width, w[0], w[1], pos, freq, slots, *caches, tokens, hq, hk, d, rot, 16, 1e-6)
        if fp8:
            atlas.qkv_norm_rope_cache_write_fp8(*args, 30.0, 50.0)
        else:
            atlas.qkv_norm_rope_cache_write(*args)
    torch.cuda.synchronize()
    at = (n_rows - tokens) * row
    assert at > 1 << 32
    for far, near in zip(sides, small):
        assert near[:tokens * row].any() and torch.equal(far[at:at + tokens * row], near[:tokens * row])


def test_page_copies(cuda, atlas, sides):
    """A fork of a part-filled page and a compaction, pages of 1 MB."""
    torch, page_bytes, page = cuda, 1_000_000 // 256 * 256, 16
    n_pages = BYTES // page_bytes
    a, b, free = n_pages - 2, n_pages - 1, n_pages - 5
    assert free * page_bytes > 1 << 32
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    for t in sides:
        t[free * page_bytes:n_pages * page_bytes] = torch.randint(0, 256, ((n_pages - free) * page_bytes,), generator=g, dtype=torch.uint8, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    bases = torch.tensor([t.data_ptr() for t in sides], dtype=torch.int64, device="cuda")
    ref = torch.ones(n_pages, **i32)
    ref[free] = 0
    table = torch.full((2, 4), -1, **i32)
    table[0, :2] = torch.tensor([a, b])
    seq_len = torch.tensor([20, 0], **i32)
    desc = atlas.make_cache_desc(bases=bases, n_bases=2, page_bytes=page_bytes, n_pages=n_pages, block_size=page, refcount=ref, block_table=table, table_stride=4,
                                 seq_len=seq_len, n_seqs=2)
    ws = torch.empty(atlas.cache_ws_bytes(desc, 2), dtype=torch.uint8, device="cuda")
    desc.ws, desc.ws_bytes = ws.data_ptr(), ws.numel()
    before = [t[free * page_bytes:n_pages * page_bytes].clone().view(-1, page_bytes) for t in sides]
    status = torch.full((1,), 9, **i32)
    atlas.cache_fork(desc, torch.tensor([0], **i32), torch.tensor([1], **i32), 1, status)
    torch.cuda.synchronize()
    assert status.tolist() == [0] and table[1].tolist()[:2] == [a, free] and seq_len.tolist() == [20, 20] and int(ref[a]) == 2 and int(ref[free]) == 1
    part = page_bytes // page * 4
    for t, was in zip(sides, before):
        now = t[free * page_bytes:n_pages * page_bytes].view(-1, page_bytes)
        assert torch.equal(now[0, :part], was[-1, :part]) and torch.equal(now[0, part:], was[0, part:]) and torch.equal(now[1:], was[1:])
    ref[:] = 0
    ref[free], ref[a], ref[b] = 1, 2, 1
    pages_were = [t[free * page_bytes:n_pages * page_bytes].clone().view(-1, page_bytes) for t in sides]
    page_map, n_used = torch.full((n_pages,), 9, **i32), torch.zeros(1, **i32)
    atlas.cache_compact(desc, ref, table, page_map, n_used)
    torch.cuda.synchronize()
    assert n_used.item() == 3 and table[:, :2].tolist() == [[1, 2], [1, 0]] and ref[:4].tolist() == [1, 2, 1, 0] and np.count_nonzero(ref.cpu().numpy()) == 3
    for t, was in zip(sides, pages_were):
        now = t[:3 * page_bytes].view(-1, page_bytes)
        assert torch.equal(now[0], was[0]) and torch.equal(now[1], was[a - free]) and torch.equal(now[2], was[b - free])
    assert atlas.device_status() == 0
