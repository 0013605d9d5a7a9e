"""Paged attention over E4M3 caches at the ends of its numbers' ranges."""
import math

import pytest

from attention_util import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[(1, 700), (1, 3)], [(1, 9000)], [(3, 100), (2, 33)], [(50, 300), (9, 5)]], ids=["decode", "long", "few", "chunk"])
@pytest.mark.parametrize("scale,k_scale,q_exp", [(1e-30, 1e-30, 0), (None, 1e-9, -110), (1e-38, 1e-3, -60)])
def test_factors_below_what_fp32_holds(cuda, atlas, lens, scale, k_scale, q_exp):
    """Scores that are nothing beside the softmax's resolution: every key that is seen has the same weight."""
    b = Batch(cuda, atlas, lens, 8, 2, 128, 16, True, seed=1, scale=scale)
    b.k_scale = k_scale
    b.q *= 2.0 ** q_exp
    atlas.paged_attention(b.desc())
    b.check()


@pytest.mark.parametrize("new,seqs,heads,d,sinks", [(1, 230, 4, 64, (0, 32, 64, 96)), (1, 230, 4, 128, (0, 32, 64, 96)), (1, 230, 4, 256, (0, 16, 32, 48)), (1, 230, 16, 128, (0, 32, 64, 96)),
                                                   (40, 1, 1, 64, (0,)), (40, 1, 1, 128, (0,)), (40, 1, 1, 256, (0,)), (40, 1, 1, 128, (100000,))])
def test_many_weights_far_below_the_largest(cuda, atlas, new, seqs, heads, d, sinks):
    """One key (of each warp's, where warps have keys of their own) outweighs any other by 2^25.4, and has zeros for values: what the output is comes
    from the 2^18 others.  Without scratch, so that the keys are not shared out to many SMs, each with a largest weight of its own.

    A weight is rounded to FP16 at 2^7 times its share of the largest: off by 2^-11 of itself or 2^-32 of the largest.  The rest as in
    attention_util: scores off by (d + 4) 2^-23 of themselves, 2^-21 an exponential, 2^-24 a key for the sum, 2^-23 for the products."""
    torch = cuda
    n, page, score = 1 << 18, 64, 17.625
    k = torch.zeros((n, 1, d), dtype=torch.uint8, device="cuda")
    v = torch.full((n, 1, d), 0x38, dtype=torch.uint8, device="cuda")                 # 1.0
    for at in sinks:
        k[at, 0, 0] = 0x58                                                            # 16.0
        v[at] = 0
    assert torch.tensor([0x38, 0x58], dtype=torch.uint8).view(torch.float8_e4m3fn).tolist() == [1.0, 16.0]
    q = torch.zeros((new * seqs, heads * d), dtype=torch.bfloat16, device="cuda")
    q.view(-1, heads, d)[:, :, 0] = score / 16.0
    out = torch.empty_like(q)
    lse = torch.empty((new * seqs, heads), dtype=torch.float32, device="cuda")
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").repeat(seqs, 1)
    cu = (torch.arange(seqs + 1, device="cuda") * new).int()
    kv = torch.full((seqs,), n, dtype=torch.int32, device="cuda")
    atlas.paged_attention(atlas.make_attention_desc(
        q=q, out=out, lse=lse, k_cache=k, v_cache=v, block_table=table, cu_q=cu, kv_len=kv, n_seqs=seqs, n_tokens=new * seqs, max_q_len=new, max_kv_len=n,
        n_pages=n // page, block_size=page, table_stride=n // page, q_heads=heads, kv_heads=1, head_dim=d, softmax_scale=1.0, cache_dtype=atlas.CACHE_E4M3))
    torch.cuda.synchronize()
    shape = atlas.last_attention_shape()
    assert shape["whole_items"] and (new > 1 or shape["ctas"] == seqs) and shape["block_rows"] == ((8 if heads <= 8 else 16) if new == 1 else 128 if d == 256 else 256)
    err = 1.01 * score * (d + 4) * 2.0 ** -23 + 2.0 ** -21 + n * 2.0 ** -24
    got, got_l = out.view(seqs, new, heads, d).double(), lse.view(seqs, new, heads).double()
    for i in range(new):
        seen = n - new + i + 1
        large = len(sinks) * math.exp(score)
        total = seen - len(sinks) + large
        want = (seen - len(sinks)) / total
        tol = want * (2 * err + 2.0 ** -11 + n * 2.0 ** -23 + 2.0 ** -8) + n * 2.0 ** -32 * math.exp(score) / total
        assert tol < want / 8
        assert ((got[:, i] - want).abs() <= tol).all(), (i, got[:, i].min().item(), got[:, i].max().item(), want, tol)
        assert ((got_l[:, i] - math.log(total)).abs() <= 2 * err + 2.0 ** -22 * (1 + math.log(total))).all()
    assert atlas.device_status() == 0
