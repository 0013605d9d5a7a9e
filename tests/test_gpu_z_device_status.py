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


@pytest.mark.parametrize("chunk", [1, 60], ids=["decode", "chunk"])
@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
def test_a_skipped_sequence_leaves_no_record(cuda, atlas, chunk, fp8):
    """Entries without new tokens pad a captured batch: their lengths and tables may hold anything."""
    lens = [(chunk, 500), (0, 0), (chunk, 70), (0, 0), (0, 0)]
    b = Batch(cuda, atlas, lens, 8, 2, 64, 16, fp8, seed=2)
    b.kv[1], b.kv[3], b.kv[4] = 0x7FFFFFFF, b.stride * 16 + 1, -1
    desc = b.desc()
    atlas.paged_attention(desc)
    b.check()                                          # (and the status is 0)
    b.kv[0] = 0x7FFFFFFF                               # one that has new tokens is recorded
    b.table[0] = b.table[0, 0]
    atlas.paged_attention(desc)
    cuda.cuda.synchronize()
    assert atlas.device_status() == 5 and atlas.device_status() == 0
