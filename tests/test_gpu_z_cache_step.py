"""A server's steps over the paged cache through the public calls: pages are taken, the QKV consumer writes into them, the attention
reads them, sequences are forked, extended, freed, and the pool is compacted — against attention over each sequence's own history."""
import math

import pytest

pytestmark = pytest.mark.gpu

HQ, HK, D, PAGE, STRIDE, N_PAGES = 8, 2, 128, 16, 12, 90
K_INV, V_INV = 40.0, 60.0


class Server:
    def __init__(self, torch, atlas, fp8, seed):
        self.torch, self.atlas, self.fp8 = torch, atlas, fp8
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)
        kind = dict(dtype=torch.float8_e4m3fn if fp8 else torch.bfloat16, device="cuda")
        self.caches = torch.zeros((2, N_PAGES, PAGE, HK, D), **kind)
        n_seqs = self.n_seqs = 10
        i32 = dict(dtype=torch.int32, device="cuda")
        self.ref, self.table, self.lens = torch.zeros(N_PAGES, **i32), torch.full((n_seqs, STRIDE), -1, **i32), torch.zeros(n_seqs, **i32)
        self.bases = torch.tensor([c.data_ptr() for c in self.caches], dtype=torch.int64, device="cuda")
        self.pages = atlas.make_cache_desc(bases=self.bases, n_bases=2, page_bytes=PAGE * HK * D * (1 if fp8 else 2), n_pages=N_PAGES, block_size=PAGE,
                                           refcount=self.ref, block_table=self.table, table_stride=STRIDE, seq_len=self.lens, n_seqs=n_seqs)
        self.ws = torch.empty(atlas.cache_ws_bytes(self.pages, n_seqs), dtype=torch.uint8, device="cuda")
        self.pages.ws, self.pages.ws_bytes = self.ws.data_ptr(), self.ws.numel()
        self.w = [(torch.randn(D, generator=self.g, device="cuda") * 0.1).to(torch.bfloat16) for _ in range(2)]
        self.freq = (1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)).float()
        self.history = {s: ([], []) for s in range(n_seqs)}             # K and V as the cache holds them

    def i32(self, v):
        return self.torch.tensor(list(v), dtype=self.torch.int32, device="cuda")

    def extend(self, n_new):
        """n_new: {sequence: tokens}.  Returns q and out of the new tokens; checks the attention."""
        torch, atlas = self.torch, self.atlas
        seqs, total = list(n_new), sum(n_new.values())
        slots = torch.empty(total, dtype=torch.int64, device="cuda")
        status = self.i32([9] * len(seqs))
        atlas.cache_append(self.pages, self.i32(seqs), self.i32(n_new.values()), len(seqs), slots, total, status)
        assert status.tolist() == [0] * len(seqs)
        lens = self.lens[torch.tensor(seqs, device="cuda")].contiguous()
        pos = torch.cat([torch.arange(n - k, n) for n, k in zip(lens.tolist(), n_new.values())]).to(torch.int32).cuda()
        width = (HQ + 2 * HK) * D
        qkv = torch.randn((total, width), generator=self.g, device="cuda").to(torch.bfloat16)
        base = qkv.data_ptr()
        write = atlas.qkv_norm_rope_cache_write_fp8 if self.fp8 else atlas.qkv_norm_rope_cache_write
        write(base, base + 2 * HQ * D, base + 2 * (HQ + HK) * D, width, width, self.w[0], self.w[1], pos, self.freq, slots, self.caches[0], self.caches[1], total, HQ, HK,
              D, D, PAGE, 1e-6, *((K_INV, V_INV) if self.fp8 else ()))
        out = torch.empty((total, HQ * D), dtype=torch.bfloat16, device="cuda")
        cu = self.i32([0] + list(torch.tensor(list(n_new.values())).cumsum(0)))
        rows = self.table[torch.tensor(seqs, device="cuda")].contiguous()
        desc = atlas.make_attention_desc(q=qkv, out=out, k_cache=self.caches[0], v_cache=self.caches[1], block_table=rows, cu_q=cu, kv_len=lens, n_seqs=len(seqs),
                                         n_tokens=total, max_q_len=max(n_new.values()), max_kv_len=STRIDE * PAGE, n_pages=N_PAGES, block_size=PAGE, table_stride=STRIDE,
                                         q_heads=HQ, kv_heads=HK, head_dim=D, q_row_stride=width, softmax_scale=1 / math.sqrt(D),
                                         cache_dtype=atlas.CACHE_E4M3 if self.fp8 else atlas.CACHE_BF16, k_scale=1 / K_INV if self.fp8 else 1.0,
                                         v_scale=1 / V_INV if self.fp8 else 1.0)
        ws = torch.empty(max(atlas.attention_ws_bytes(desc), 16), dtype=torch.uint8, device="cuda")
        desc.ws, desc.ws_bytes = ws.data_ptr(), ws.numel()
        atlas.paged_attention(desc)
        torch.cuda.synchronize()
        # what the writer put into the slots joins each sequence's history, and the attention is that history's
        at = 0
        for s, k in n_new.items():
            mine = slots[at:at + k]
            for side in range(2):
                self.history[s][side].append(self.caches[side].view(-1, HK, D)[mine].double())
            keys, values = (torch.cat(h) for h in self.history[s])
            if self.fp8:
                keys, values = keys / K_INV, values / V_INV
            n = keys.shape[0]
            for i in range(k):
                for h in range(HQ):
                    q = qkv[at + i, h * D:(h + 1) * D].double()
                    seen = n - k + i + 1
                    p = torch.softmax(keys[:seen, h // 4] @ q / math.sqrt(D), 0)
                    want, size = p @ values[:seen, h // 4], p @ values[:seen, h // 4].abs()
                    # P's rounding and the output's, 2^-8 each, and 2^-12 for the FP32 sums
                    assert ((out[at + i, h * D:(h + 1) * D].double() - want).abs() <= size * (2.0 ** -8 + 2.0 ** -12) + want.abs() * 2.0 ** -8).all()
            at += k
        return desc, out

    def fork(self, src, dst):
        status = self.i32([9] * len(src))
        self.atlas.cache_fork(self.pages, self.i32(src), self.i32(dst), len(src), status)
        assert status.tolist() == [0] * len(src)
        for a, b in zip(src, dst):
            self.history[b] = (list(self.history[a][0]), list(self.history[a][1]))

    def free(self, seqs):
        self.atlas.cache_free(self.pages, self.i32(seqs), len(seqs))
        for s in seqs:
            self.history[s] = ([], [])


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "e4m3"])
def test_steps(cuda, atlas, fp8):
    s = Server(cuda, atlas, fp8, seed=21)
    s.extend({0: 37, 1: 100, 2: 1})
    s.extend({0: 1, 1: 1, 2: 1})
    s.fork([0, 1, 1], [5, 6, 7])
    s.extend({5: 4, 6: 2, 7: 20, 1: 1})
    s.free([1, 0])
    s.fork([7], [0])
    s.extend({0: 1, 5: 1, 2: 30, 8: 16})
    page_map, used = cuda.empty_like(s.ref), s.i32([0])
    atlas.cache_compact(s.pages, s.ref, s.table, page_map, used)
    assert used.item() == int((s.ref > 0).sum()) and int((s.ref[used.item():] != 0).sum()) == 0
    s.extend({0: 1, 2: 3, 5: 1, 6: 1, 7: 1, 8: 1})
    s.free([0, 2, 5, 6, 7, 8])
    assert int(s.ref.abs().sum()) == 0 and atlas.device_status() == 0
