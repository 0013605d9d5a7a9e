"""Refusals of calls around the paged cache that a kernel could not carry out, and what their scratch is asked for: no device is touched."""
import pytest

OK, ALIGN = 0, -3
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
