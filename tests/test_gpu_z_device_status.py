"""The device status over both halves of the library: what the linear path's kernels record and what the cache operators' do."""
import pytest

from attention_util import Batch

pytestmark = pytest.mark.gpu


def test_neither_record_hides_the_other(cuda, atlas):
    assert atlas.device_status() == 0
    b = Batch(cuda, atlas, [(1, 40), (1, 7)], 4, 2, 64, 16, seed=1)
    b.table[0, 1] = b.n_pages
    desc = b.desc()
    for first in ("attention", "wait"):
        for what in (first, "wait" if first == "attention" else "attention"):
            if what == "attention":
                atlas.paged_attention(desc)
                cuda.cuda.synchronize()
            else:
                atlas.selftest_bounded_wait(1_000_000)
        assert atlas.device_status(clear=False) == 0x100 and atlas.device_status(clear=False) == 0x100
        assert atlas.device_status() == 0x100          # an expired wait, of the linear path's kernels
        assert atlas.device_status(clear=False) == 4   # a page that is not of the pool, of the attention's
        assert atlas.device_status() == 4
        assert atlas.device_status() == 0
