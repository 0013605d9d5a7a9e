"""Pages of the paged cache between two steps, against a model of them in Python: every table, count, slot, status and byte."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class Model:
    """The operators' definitions, one entry and one page at a time."""

    def __init__(self, page, ref, table, lens, caches):
        self.page, self.ref, self.table, self.lens, self.caches = page, ref.copy(), table.copy(), lens.copy(), caches.copy()

    def held(self, n):
        return -(-int(n) // self.page)

    def free_pages(self):
        return list(np.flatnonzero(self.ref == 0))

    def free(self, seqs):
        for s in seqs:
            if not 0 <= s < len(self.lens):
                continue
            for k in range(self.held(self.lens[s])):
                self.ref[self.table[s, k]] -= 1
                self.table[s, k] = -1
            self.lens[s] = 0

    def fork(self, src, dst):
        status, free, given = [], self.free_pages(), 0
        before, seen = self.lens.copy(), set()
        for a, b in zip(src, dst):
            ok = 0 <= a < len(before) and 0 <= b < len(before) and a != b and b not in seen and before[b] == 0
            if 0 <= b < len(before):
                seen.add(b)
            if not ok:
                status.append(-1)
                continue
            full, rest = divmod(int(before[a]), self.page)
            if rest:
                given += 1
                if given > len(free):
                    status.append(-5)
                    continue
            for k in range(full):
                self.table[b, k] = self.table[a, k]
                self.ref[self.table[a, k]] += 1
            if rest:
                to = free[given - 1]
                self.ref[to] = 1
                self.table[b, full] = to
                self.caches[:, to, :rest] = self.caches[:, self.table[a, full], :rest]
            self.lens[b] = before[a]
            status.append(0)
        return status

    def append(self, seqs, n_new, max_tokens):
        status, slots, free, given, seen = [], [], self.free_pages(), 0, set()
        for s, n in zip(seqs, n_new):
            first = len(slots)
            ok = 0 <= s < len(self.lens) and s not in seen and n >= 0
            if 0 <= s < len(self.lens):
                seen.add(s)
            n = max(n, 0)
            slots += [-1] * n
            if not ok:
                status.append(-1)
                continue
            have, want = self.held(self.lens[s]), self.held(self.lens[s] + n)
            if self.lens[s] + n > self.table.shape[1] * self.page or first + n > max_tokens:
                status.append(-5)
                continue
            given += want - have
            if want > have and given > len(free):
                status.append(-5)
                continue
            pages = free[given - (want - have):given] if want > have else []
            self.table[s, have:want] = pages
            self.ref[pages] = 1
            for k in range(n):
                pos = int(self.lens[s]) + k
                slots[first + k] = int(self.table[s, pos // self.page]) * self.page + pos % self.page
            self.lens[s] += n
            status.append(0)
        return status, (slots + [-1] * max_tokens)[:max_tokens]

    def compact(self):
        used = np.flatnonzero(self.ref > 0)
        u = len(used)
        page_map = np.where(self.ref > 0, np.arange(len(self.ref)), -1).astype(np.int32)
        moved, holes = [p for p in used if p >= u], [p for p in range(u) if self.ref[p] == 0]
        for a, b in zip(moved, holes):
            page_map[a] = b
            self.ref[b], self.ref[a] = self.ref[a], 0
            self.caches[:, b] = self.caches[:, a]
        for s in range(len(self.lens)):
            for k in range(self.held(self.lens[s])):
                self.table[s, k] = page_map[self.table[s, k]]
        return page_map, u


class Pool:
    def __init__(self, torch, atlas, lens, n_pages, page, stride, token=32, layers=3, more=0, seed=0, n_max=64, dtype=np.int16):
        rng = np.random.default_rng(seed)
        perm, at = rng.permutation(n_pages), 0
        table = np.full((len(lens) + more, stride), -1, np.int32)
        ref = np.zeros(n_pages, np.int32)
        for i, n in enumerate(lens):
            k = -(-n // page)
            table[i, :k] = perm[at:at + k]
            at += k
        ref[perm[:at]] = 1
        caches = rng.integers(-2 ** 15, 2 ** 15, (2 * layers, n_pages, page, token)).astype(dtype)
        self.torch, self.atlas, self.n_max = torch, atlas, n_max
        self.model = Model(page, ref, table, np.array(list(lens) + [0] * more, np.int32), caches)
        m = self.model
        self.ref, self.table, self.lens, self.caches = (torch.from_numpy(x.copy()).cuda() for x in (m.ref, m.table, m.lens, m.caches))
        self.bases = torch.tensor([c.data_ptr() for c in self.caches], dtype=torch.int64, device="cuda")
        self.desc = atlas.make_cache_desc(bases=self.bases, n_bases=2 * layers, page_bytes=page * token * caches.itemsize, n_pages=n_pages, block_size=page,
                                          refcount=self.ref, block_table=self.table, table_stride=stride, seq_len=self.lens, n_seqs=len(m.lens))
        self.ws = torch.full((atlas.cache_ws_bytes(self.desc, n_max),), 0xA5, dtype=torch.uint8, device="cuda")
        self.desc.ws, self.desc.ws_bytes = self.ws.data_ptr(), self.ws.numel()

    def i32(self, v):
        return self.torch.tensor(list(v), dtype=self.torch.int32, device="cuda")

    def check(self):
        self.torch.cuda.synchronize()
        m = self.model
        for name, got, want in (("lens", self.lens, m.lens), ("ref", self.ref, m.ref), ("table", self.table, m.table), ("caches", self.caches, m.caches)):
            assert np.array_equal(got.cpu().numpy(), want), name

    def free(self, seqs):
        self.atlas.cache_free(self.desc, self.i32(seqs), len(seqs))
        self.model.free(seqs)

    def fork(self, src, dst):
        st = self.i32([9] * len(src))
        self.atlas.cache_fork(self.desc, self.i32(src), self.i32(dst), len(src), st)
        want = self.model.fork(src, dst)
        assert st.tolist() == want
        return want

    def append(self, seqs, n_new, spare=5, max_tokens=None):
        most = sum(max(n, 0) for n in n_new) + spare if max_tokens is None else max_tokens
        st, slots = self.i32([9] * len(seqs)), self.torch.full((most + 2,), 12345, dtype=self.torch.int64, device="cuda")
        self.atlas.cache_append(self.desc, self.i32(seqs), self.i32(n_new), len(seqs), slots, most, st)
        want, want_slots = self.model.append(seqs, n_new, most)
        assert st.tolist() == want
        assert slots.tolist() == want_slots + [12345] * 2
        return want

    def compact(self, in_place):
        torch = self.torch
        ref, table = (self.ref, self.table) if in_place else (torch.full_like(self.ref, 7), torch.full_like(self.table, 7))
        page_map, used = torch.full_like(self.ref, 7), self.i32([7])
        self.atlas.cache_compact(self.desc, ref, table, page_map, used)
        want_map, want_used = self.model.compact()
        assert used.item() == want_used and np.array_equal(page_map.cpu().numpy(), want_map)
        if not in_place:
            self.ref.copy_(ref)
            self.table.copy_(table)


@pytest.mark.parametrize("page,token", [(16, 32), (5, 16), (1, 24), (8, 1), (24, 40)])
def test_a_life_of_a_pool(cuda, atlas, page, token):
    """Forks, appends, frees and compactions in a random order, as a server makes them."""
    rng = np.random.default_rng(page)
    lens = [int(n) for n in rng.integers(0, 9 * page + 2, 12)]
    p = Pool(cuda, atlas, lens, 12 * 10 + 60, page, 12, token=token, more=20, seed=page)
    for step in range(12):
        empty = [s for s in range(len(p.model.lens)) if p.model.lens[s] == 0]
        live = [s for s in range(len(p.model.lens)) if p.model.lens[s] > 0]
        rng.shuffle(empty)
        n = min(len(empty), int(rng.integers(1, 9)))
        p.fork([int(s) for s in rng.choice(live, n)], [int(s) for s in empty[:n]])
        seqs = [int(s) for s in rng.permutation(len(p.model.lens))[:9]]
        p.append(seqs, [int(k) for k in rng.integers(0, 2 * page + 3, 9)])
        p.free([int(s) for s in rng.permutation(live)[:4]] + [int(live[0])] * 2)
        if step % 3 == 2:
            p.compact(in_place=step % 2 == 0)
        p.check()
    assert atlas.device_status() == 0


def test_entries_that_cannot_be(cuda, atlas):
    """The same sequence twice, sequences that do not exist, targets that are not empty, a pool that runs out in the middle."""
    p = Pool(cuda, atlas, [10, 16, 33, 5], 9, 16, 4, more=4, seed=1)          # 1 + 1 + 3 + 1 pages: three are free
    assert p.fork([0, 0, 1, 2, 3, 7, 99, -1, 0], [4, 4, 0, 99, -1, 5, 5, 6, 6]) == [0, -1, -1, -1, -1, 0, -1, -1, -1]
    p.check()                                                                 # (an entry that fails has named its target all the same)
    assert p.append([0, 1, 1, 3, 5, 2, 200, 4], [3, 2, 1, 12, 0, 40, 2, -4]) == [0, 0, -1, 0, 0, -5, -1, -1]
    p.check()
    # no page is left: those that need none are served
    assert p.append([0, 1, 4, 5], [20, 1, 6, 1]) == [-5, 0, 0, -5]
    p.check()
    assert p.append([3, 0], [3, 6], max_tokens=6) == [0, -5]                  # no room for the second one's slots
    p.check()
    p.free([0, 0, 1, 2, 3, 4, 5, 6])
    p.check()
    assert (p.model.ref == 0).all()
    p.free([100])
    cuda.cuda.synchronize()
    assert atlas.device_status() == 6
    p.check()


def test_a_page_given_back_too_often(cuda, atlas):
    p = Pool(cuda, atlas, [20], 4, 16, 4, seed=2)
    p.ref.zero_()
    p.atlas.cache_free(p.desc, p.i32([0]), 1)
    cuda.cuda.synchronize()
    assert atlas.device_status() == 7 and (p.ref == 0).all() and (p.table == -1).all()


@pytest.mark.parametrize("n_pages", [1, 4095, 4097, 9000])
def test_pools_around_a_turn(cuda, atlas, n_pages):
    """Pools of less, just more and several times what the planning CTA looks at in a turn."""
    rng = np.random.default_rng(n_pages)
    most = max(1, n_pages // 2)
    lens, left = [], most
    while left > 0:
        k = int(rng.integers(1, min(left, 400) + 1))
        lens.append(8 * k - int(rng.integers(0, 8)))
        left -= k
    p = Pool(cuda, atlas, lens, n_pages, 8, 420, token=8, layers=1, more=8, seed=3)
    first = len(lens)
    if n_pages > 1:
        p.fork([0, first - 1, 0], [first, first + 1, first + 2])
        p.append([first + 3, 0, first + 4], [min(3000, n_pages), 5, 1])
        p.check()
    p.compact(in_place=False)
    p.check()
    p.compact(in_place=True)                                                # nothing is left to move
    p.check()


def test_many_entries(cuda, atlas):
    """More entries than the planning CTA has threads."""
    n = 2500
    p = Pool(cuda, atlas, [3] * 50, 6000, 4, 3, token=8, layers=1, more=n, seed=4, n_max=n)
    assert set(p.fork([i % 50 for i in range(n)], list(range(50, 50 + n)))) == {0}
    assert set(p.append(list(range(50, 50 + n)), [i % 7 for i in range(n)])) == {0}
    p.check()
    p.free(list(range(40, 2000)))
    p.check()
    p.compact(in_place=True)
    p.check()


def test_no_caches_and_no_statuses(cuda, atlas):
    p = Pool(cuda, atlas, [10, 3], 6, 4, 4, more=2, seed=5)
    p.desc.n_bases = 0
    p.desc.bases = None
    atlas.cache_fork(p.desc, p.i32([0, 1]), p.i32([2, 3]), 2)
    keep = p.model.caches.copy()
    p.model.fork([0, 1], [2, 3])
    p.model.caches = keep
    p.check()


def test_captured(cuda, atlas):
    """A captured step of frees, forks and appends goes by the state that it finds."""
    torch = cuda
    p = Pool(cuda, atlas, [10, 35, 16, 7], 60, 8, 8, more=6, seed=6)
    src, dst, n_new = p.i32([0, 1, 1, 3, 2]), p.i32([4, 5, 6, 7, 8]), p.i32([1, 2, 3, 4, 5])
    st, st2, slots = p.i32([9] * 5), p.i32([9] * 5), torch.full((20,), 5, dtype=torch.int64, device="cuda")

    def step():
        atlas.cache_free(p.desc, dst, 5)
        atlas.cache_fork(p.desc, src, dst, 5, st)
        atlas.cache_append(p.desc, dst, n_new, 5, slots, 20, st2)

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.synchronize()
    m = p.model
    for round_ in range(4):
        graph.replay()
        m.free(range(4, 9))
        assert st.tolist() == m.fork(src.tolist(), dst.tolist())
        want, want_slots = m.append(dst.tolist(), n_new.tolist(), 20)
        assert st2.tolist() == want and slots.tolist() == want_slots
        p.check()
        src.copy_(torch.roll(src, 1))
        n_new.copy_(torch.roll(n_new, 2))
