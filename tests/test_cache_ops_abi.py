"""Refusals of the operators around the paged cache and the layout of their descriptors: no device is touched."""
import ctypes as C

import pytest

OK, DIMS, WORKSPACE, ALIGN, NULL, LIMIT = 0, -1, -2, -3, -4, -5
A = 1 << 20        # an address that no call below gets as far as using


def attention_desc(atlas, **kw):
    a = dict(q=A, out=A, k_cache=A, v_cache=A, block_table=A, cu_q=A, kv_len=A, n_seqs=2, n_tokens=2, max_q_len=1, max_kv_len=100, n_pages=10, block_size=16,
             table_stride=7, q_heads=8, kv_heads=2, head_dim=128, softmax_scale=0.1)
    a.update(kw)
    return atlas.make_attention_desc(**a)


def test_descriptor_layouts(atlas):
    d = atlas.AttentionDesc
    assert d.lse.offset == 16 and d.ws.offset == 64 and d.ws_bytes.offset == 72 and d.n_seqs.offset == 80 and d.n_pages.offset == 96
    assert d.q_heads.offset == 112 and d.out_row_stride.offset == 128 and d.v_scale.offset == 140 and C.sizeof(d) == 144
    c = atlas.CacheDesc
    assert c.seq_len.offset == 24 and c.page_bytes.offset == 48 and c.n_bases.offset == 56 and c.n_seqs.offset == 72 and C.sizeof(c) == 80


@pytest.mark.parametrize("change,status", [
    (dict(head_dim=0), DIMS), (dict(head_dim=48), DIMS), (dict(head_dim=288), DIMS), (dict(kv_heads=0), DIMS), (dict(kv_heads=3), DIMS), (dict(q_heads=0), DIMS),
    (dict(block_size=0), DIMS), (dict(table_stride=0), DIMS), (dict(n_pages=0), DIMS), (dict(cache_dtype=2), DIMS), (dict(softmax_scale=0.0), DIMS),
    (dict(softmax_scale=float("nan")), DIMS), (dict(softmax_scale=float("inf")), DIMS), (dict(softmax_scale=-1.0), DIMS), (dict(k_scale=2.0), DIMS),
    (dict(cache_dtype=1, v_scale=0.0), DIMS), (dict(cache_dtype=1, k_scale=float("inf")), DIMS), (dict(q_row_stride=1022), DIMS), (dict(out_row_stride=1023), DIMS),
    (dict(n_pages=1 << 27), LIMIT), (dict(table_stride=1 << 27), LIMIT), (dict(n_tokens=1 << 29), LIMIT), (dict(n_seqs=1 << 24), LIMIT),
    (dict(q=None), NULL), (dict(out=None), NULL), (dict(k_cache=None), NULL), (dict(v_cache=None), NULL), (dict(block_table=None), NULL), (dict(cu_q=None), NULL),
    (dict(kv_len=None), NULL),
    (dict(q=A + 2), ALIGN), (dict(q_row_stride=1025), ALIGN), (dict(k_cache=A + 8), ALIGN), (dict(v_cache=A + 2), ALIGN), (dict(cu_q=A + 2), ALIGN),
    (dict(lse=A + 2), ALIGN), (dict(out=A + 1), ALIGN), (dict(ws=A + 4, ws_bytes=1 << 30), ALIGN),
])
def test_attention_refuses(atlas, change, status):
    assert atlas.lib().atlas_b200_paged_attention(C.byref(attention_desc(atlas, **change)), None) == status


def test_attention_without_work(atlas):
    L = atlas.lib()
    assert L.atlas_b200_paged_attention(None, None) == NULL
    assert L.atlas_b200_paged_attention(C.byref(attention_desc(atlas, n_seqs=0)), None) == OK
    assert L.atlas_b200_paged_attention(C.byref(attention_desc(atlas, n_tokens=0)), None) == OK
    assert L.atlas_b200_paged_attention_ws_bytes(None) == 0
    with pytest.raises(atlas.AtlasError):
        atlas.paged_attention(attention_desc(atlas, head_dim=100), stream=0)


def cache_desc(atlas, **kw):
    a = dict(bases=A, n_bases=4, page_bytes=4096, n_pages=10, block_size=16, refcount=A, block_table=A, table_stride=4, seq_len=A, n_seqs=3, ws=A, ws_bytes=1 << 20)
    a.update(kw)
    return atlas.make_cache_desc(**a)


@pytest.mark.parametrize("change,status", [
    (dict(n_pages=0), DIMS), (dict(block_size=0), DIMS), (dict(table_stride=0), DIMS), (dict(n_seqs=0), DIMS), (dict(table_stride=1 << 27), LIMIT),
    (dict(refcount=None), NULL), (dict(block_table=None), NULL), (dict(seq_len=None), NULL), (dict(ws=None), NULL), (dict(ws_bytes=100), WORKSPACE),
    (dict(refcount=A + 2), ALIGN), (dict(ws=A + 8), ALIGN),
])
def test_page_operators_refuse(atlas, change, status):
    L, d = atlas.lib(), cache_desc(atlas, **change)
    assert L.atlas_b200_cache_append(C.byref(d), A, A, 2, 8, A, None, None) == status
    assert L.atlas_b200_cache_fork(C.byref(d), A, A, 2, None, None) == status
    assert L.atlas_b200_cache_free(C.byref(d), A, 2, None) == status
    assert L.atlas_b200_cache_compact(C.byref(d), A, A, A, A, None) == status


def test_copying_operators_refuse(atlas):
    L = atlas.lib()
    for change, status in ((dict(page_bytes=0), DIMS), (dict(page_bytes=4100), DIMS), (dict(page_bytes=4104, block_size=8), DIMS), (dict(bases=None), NULL),
                           (dict(n_bases=1 << 16), LIMIT), (dict(bases=A + 4), ALIGN)):
        d = cache_desc(atlas, **change)
        assert L.atlas_b200_cache_fork(C.byref(d), A, A, 2, None, None) == status
        assert L.atlas_b200_cache_compact(C.byref(d), A, A, A, A, None) == status
    d = C.byref(cache_desc(atlas))
    assert L.atlas_b200_cache_append(d, None, A, 2, 8, A, None, None) == NULL
    assert L.atlas_b200_cache_append(d, A, A, 2, 8, None, None, None) == NULL
    assert L.atlas_b200_cache_append(d, A, A, 2, 8, A + 4, None, None) == ALIGN
    assert L.atlas_b200_cache_append(d, A, A, 2, 1 << 31, A, None, None) == LIMIT
    assert L.atlas_b200_cache_append(d, None, None, 0, 0, None, None, None) == OK
    assert L.atlas_b200_cache_fork(d, A, None, 2, None, None) == NULL
    assert L.atlas_b200_cache_fork(d, None, None, 0, None, None) == OK
    assert L.atlas_b200_cache_free(d, None, 2, None) == NULL
    assert L.atlas_b200_cache_free(d, A + 1, 2, None) == ALIGN
    assert L.atlas_b200_cache_compact(d, A, None, A, A, None) == NULL
    assert L.atlas_b200_cache_free(None, A, 2, None) == NULL


def test_fp8_writer_refuses(atlas):
    f = atlas.lib().atlas_b200_qkv_norm_rope_cache_write_fp8

    def call(k_inv=1.0, v_inv=1.0, kc=A, vc=A, d=128, stride=1024):
        return f(A, A, A, stride, stride, A, A, A, A, A, kc, vc, 0 if (k_inv, v_inv, kc, vc, d, stride) == (1.0, 1.0, A, A, 128, 1024) else 4, 4, 2, d, 64, 16,
                 1e-6, 1.0, 1, k_inv, v_inv, None)
    assert call() == OK
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        assert call(k_inv=bad) == DIMS and call(v_inv=bad) == DIMS
    assert call(kc=A + 1) == ALIGN and call(vc=A + 2) == ALIGN and call(kc=None) == NULL and call(d=257) == DIMS and call(stride=1) == DIMS
