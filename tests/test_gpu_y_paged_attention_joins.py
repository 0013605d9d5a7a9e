"""Paged attention whose items are cut into many pieces: the join of blocks with fewer rows than it has CTAs for them."""
import math

import pytest

from attention_util import Batch

pytestmark = pytest.mark.gpu

BOTH = pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])


@BOTH
@pytest.mark.parametrize("new,heads,kv_heads,d,block_rows", [(1, 4, 1, 128, 8), (1, 1, 1, 64, 8), (3, 4, 2, 128, 8), (3, 3, 1, 256, 16), (65, 4, 1, 128, 256), (129, 2, 1, 128, 256),
                                                             (65, 2, 1, 256, 128)])
def test_many_pieces_of_few_rows(cuda, atlas, new, heads, kv_heads, d, block_rows, fp8):
    """More than eight pieces to an item, blocks (or last blocks) of one to seven rows, and a NaN among the values that the last token alone
    sees: it reaches that token's rows and no other, of this sequence or behind it."""
    torch = cuda
    n = 40000
    b = Batch(cuda, atlas, [(new, n), (1, 3)], heads, kv_heads, d, 16, fp8, seed=new + d)
    desc = b.desc()
    atlas.paged_attention(desc)
    shape = atlas.last_attention_shape()
    assert shape["block_rows"] == block_rows and not shape["whole_items"]
    assert shape["ctas"] >= 10 * kv_heads * -(-new * (heads // kv_heads) // block_rows)
    b.check()
    out, lse, tol, tol_l = b.exact()
    at = b.slots(0, n)[n - 1]
    if fp8:
        b.v.view(torch.uint8)[at, 0, 5] = 0x7F
    else:
        b.v[at, 0, 5] = math.nan
    b.out.fill_(77.0)
    b.lse.fill_(77.0)
    atlas.paged_attention(desc)
    torch.cuda.synchronize()
    odd = torch.isnan(b.out.float()).view(b.out.shape[0], heads, d)
    want = torch.zeros_like(odd)
    want[new - 1, :heads // kv_heads, 5] = True
    assert torch.equal(odd, want)
    # the rows that the NaN was masked in are computed again, in another order and with weights in FP32: within the same bounds
    keep = ~want[:b.rows]
    assert ((b.out[:b.rows].double().view(out.shape) - out).abs() <= tol)[keep].all()
    assert ((b.lse[:b.rows].double() - lse).abs() <= tol_l).all()
    assert (b.out[b.rows:] == 77.0).all() and (b.lse[b.rows:] == 77.0).all() and atlas.device_status() == 0


@BOTH
@pytest.mark.parametrize("new,kv", [(1, 5000), (40, 3000)])
def test_one_scratch_buffer_over_batch_sizes(cuda, atlas, new, kv, fp8):
    """A buffer as the largest batch asks for it serves the smaller ones, although these are cut into more pieces."""
    torch = cuda
    largest = Batch(cuda, atlas, [(new, kv)] * 20, 16, 4, 128, 16, fp8, seed=1).desc(ws=False)
    n = atlas.attention_ws_bytes(largest)
    ws = torch.full((n // 4,), math.nan, dtype=torch.float32, device="cuda")
    cut = 0
    for seqs in (20, 16, 8, 3, 1):
        b = Batch(cuda, atlas, [(new, kv - 7 * i) for i in range(seqs)], 16, 4, 128, 16, fp8, seed=seqs)
        d = b.desc(ws=False)
        d.ws, d.ws_bytes = ws.data_ptr(), n
        assert atlas.attention_ws_bytes(d) <= n
        atlas.paged_attention(d)
        b.check()
        cut += not atlas.last_attention_shape()["whole_items"]
    assert cut
