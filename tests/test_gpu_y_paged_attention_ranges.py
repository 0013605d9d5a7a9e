"""Paged attention over E4M3 caches at the ends of its numbers' ranges."""
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
