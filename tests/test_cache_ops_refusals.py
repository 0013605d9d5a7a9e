"""Refusals of calls around the paged cache that a kernel could not carry out, and what their scratch is asked for: no device is touched."""
import itertools

import pytest

OK, DIMS, ALIGN = 0, -1, -3
A = 1 << 20        # an address that no call below gets as far as using


@pytest.mark.parametrize("d,rot", [(128, 128), (256, 256), (128, 64), (64, 64), (96, 32)])
def test_bf16_writer_refuses_what_its_words_cannot_reach(atlas, d, rot):
    """K and V pairs are stored as 32-bit words, whichever part of the head is rotated."""
    f = atlas.lib().atlas_b200_qkv_norm_rope_cache_write

    def call(tokens=4, **kw):
        a = dict(q=A, k_in=A, v_in=A, qw=A, kw=A, kc=A, vc=A, stride=1024)
        a.update(kw)
        return f(a["q"], a["k_in"], a["v_in"], a["stride"], a["stride"], a["qw"], a["kw"], A, A, A, a["kc"], a["vc"], tokens, 4, 2, d, rot, 16, 1e-6, 1.0, 1, None)
    assert call(tokens=0) == OK
    for which in ("q", "k_in", "v_in", "qw", "kw", "kc", "vc"):
        assert call(**{which: A + 2}) == ALIGN, which
    assert call(stride=1025) == ALIGN


def _scratch(atlas, n_seqs, new, kv, heads=32, kv_heads=8, d=128, fp8=False, page=16):
    desc = atlas.make_attention_desc(q=None, out=None, k_cache=None, v_cache=None, block_table=None, cu_q=None, kv_len=None, n_seqs=n_seqs, n_tokens=n_seqs * new,
                                     max_q_len=new, max_kv_len=kv, n_pages=1 << 16, block_size=page, table_stride=1 << 14, q_heads=heads, kv_heads=kv_heads,
                                     head_dim=d, softmax_scale=0.1, cache_dtype=int(fp8))
    return atlas.attention_ws_bytes(desc)


@pytest.mark.parametrize("heads,kv_heads,d,fp8,page", [(32, 8, 128, False, 16), (32, 8, 128, True, 16), (8, 2, 64, False, 5), (12, 4, 96, True, 24), (16, 1, 256, False, 16),
                                                       (16, 2, 256, True, 7), (5, 5, 32, False, 1)])
def test_scratch_of_the_largest_batch_does_for_all(atlas, heads, kv_heads, d, fp8, page):
    """Fewer sequences, tokens or cached ones never ask for more."""
    seqs, new, kv = (1, 2, 4, 8, 16, 18, 32, 64, 300), (1, 2, 3, 5, 8, 9, 17, 64, 700), (1, 64, 200, 257, 300, 600, 4096, 100000)
    size = {k: _scratch(atlas, *k, heads, kv_heads, d, fp8, page) for k in itertools.product(seqs, new, kv)}
    for axis, values in enumerate((seqs, new, kv)):
        for k, n in size.items():
            at = values.index(k[axis])
            if at:
                less = k[:axis] + (values[at - 1],) + k[axis + 1:]
                assert size[less] <= n, (less, k)
    assert size[1, 1, 1] == 0                                  # one tile: nothing is ever cut


def test_scratch_is_that_of_the_kernel_that_runs(atlas):
    """Single tokens of four heads never take the tcgen05 form, whose pieces are thirty times as large."""
    decode, chunk = _scratch(atlas, 8, 1, 4096), _scratch(atlas, 8, 64, 4096)
    assert 0 < decode < 4 << 20 < 16 << 20 < chunk


@pytest.mark.parametrize("scale,k_scale,fp8", [(1e30, 1e30, True), (3e38, 1.0, False), (1e20, 3e18, True)])
def test_scales_whose_product_overflows(atlas, scale, k_scale, fp8):
    desc = atlas.make_attention_desc(q=A, out=A, k_cache=A, v_cache=A, block_table=A, cu_q=A, kv_len=A, n_seqs=2, n_tokens=2, max_q_len=1, max_kv_len=100, n_pages=10,
                                     block_size=16, table_stride=7, q_heads=8, kv_heads=2, head_dim=128, softmax_scale=scale, k_scale=k_scale, cache_dtype=int(fp8))
    with pytest.raises(atlas.AtlasError) as refused:
        atlas.paged_attention(desc, stream=0)
    assert refused.value.status == DIMS
