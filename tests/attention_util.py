"""A paged batch for the attention's tests, and the attention itself in 64 bits with the bound that its FP32 / BF16 computation keeps."""
import math

import numpy as np


class Batch:
    """Sequences of (new tokens, cached tokens) over a paged cache whose other places hold NaN, with table entries behind a
    sequence's last page that name no page."""

    def __init__(self, torch, atlas, lens, heads, kv_heads, d, page, fp8=False, seed=0, sharp=2.0, pad_rows=3, q_extra=0, scale=None):
        self.torch, self.atlas, self.lens, self.fp8 = torch, atlas, list(lens), fp8
        self.heads, self.kv_heads, self.d, self.page = heads, kv_heads, d, page
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        n_pages = sum(-(-kv // page) for _, kv in lens) + 5
        self.n_pages = n_pages
        self.stride = max([-(-kv // page) for _, kv in lens] + [1]) + 1
        perm, at = rng.permutation(n_pages), 0
        table = np.full((len(lens), self.stride), 0x7FFFFFF0, np.int32)
        for i, (_, kv) in enumerate(lens):
            k = -(-kv // page)
            table[i, :k] = perm[at:at + k]
            at += k
        self.table_np = table
        self.cu_np = np.concatenate([[0], np.cumsum([q for q, _ in lens])]).astype(np.int32)
        rows = self.rows = int(self.cu_np[-1])
        self.q_stride = heads * d + q_extra
        self.q = (torch.randn((rows + pad_rows, self.q_stride), generator=g, device="cuda") * sharp).to(torch.bfloat16)
        shape = (n_pages * page, kv_heads, d)
        k, v = (torch.randn(shape, generator=g, device="cuda") for _ in range(2))
        self.k_scale = self.v_scale = 1.0
        if fp8:
            self.k_scale, self.v_scale = 0.0625, 0.03125
            k, v = ((t / s).clamp(-448, 448).to(torch.float8_e4m3fn) for t, s in ((k, self.k_scale), (v, self.v_scale)))
        else:
            k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
        used = np.zeros(n_pages * page, bool)
        for i, (_, kv) in enumerate(lens):
            used[self.slots(i, kv)] = True
        stale = torch.from_numpy(~used).cuda()
        for t in (k, v):
            if fp8:
                t.view(torch.uint8)[stale] = 0x7F
            else:
                t[stale] = math.nan
        self.k, self.v = k, v
        self.table, self.cu = torch.from_numpy(table).cuda(), torch.from_numpy(self.cu_np).cuda()
        self.kv = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda")
        self.out = torch.full((rows + pad_rows, heads * d), 77.0, dtype=torch.bfloat16, device="cuda")
        self.lse = torch.full((rows + pad_rows, heads), 77.0, dtype=torch.float32, device="cuda")
        self.scale = scale or 1.0 / math.sqrt(d)

    def slots(self, i, n):
        pos = np.arange(n)
        return self.table_np[i, pos // self.page].astype(np.int64) * self.page + pos % self.page

    def desc(self, ws=True, lse=True, **kw):
        a = dict(q=self.q, out=self.out, lse=self.lse if lse else None, k_cache=self.k, v_cache=self.v, block_table=self.table, cu_q=self.cu, kv_len=self.kv,
                 n_seqs=len(self.lens), n_tokens=self.rows, max_q_len=max(q for q, _ in self.lens), max_kv_len=max(kv for _, kv in self.lens),
                 n_pages=self.n_pages, block_size=self.page, table_stride=self.stride, q_heads=self.heads, kv_heads=self.kv_heads, head_dim=self.d,
                 softmax_scale=self.scale, cache_dtype=self.atlas.CACHE_E4M3 if self.fp8 else self.atlas.CACHE_BF16, k_scale=self.k_scale,
                 v_scale=self.v_scale, q_row_stride=self.q_stride)
        a.update(kw)
        d = self.atlas.make_attention_desc(**a)
        n = self.atlas.attention_ws_bytes(d)
        if ws and n:
            self.ws = self.torch.full((n // 4 + 4,), math.nan, dtype=self.torch.float32, device="cuda")   # scratch holds nothing
            d.ws, d.ws_bytes = self.ws.data_ptr(), n
        return d

    def exact(self):
        """(out, lse, bound of out, bound of lse) in float64, [rows, heads, d] and [rows, heads].

        The kernels' arithmetic: scores are FP32 sums of d products of BF16 / FP16 values, exact themselves, so a score is off by at most
        d 2^-23 times the sum of the products' magnitudes (2^-23: tensor cores may cut off instead of rounding), and a few 2^-24 of itself
        for its factor; E4M3 caches: Q in FP16 is off by 2^-39 of the row's largest value, which the same bound covers.  exp2 is off by
        2^-21.  A weight and the sum of weights are so off by a factor of 1 + e each, e = 1.01 (score's error) + 2^-21 + (keys) 2^-24.
        Weights are then rounded to BF16 (2^-8) or FP16 (2^-11, or 2^-25 of the largest weight where that is more), products are added in
        FP32 (keys 2^-23 of the sum of magnitudes), and the output is rounded to BF16 (2^-8)."""
        torch, g, d = self.torch, self.heads // self.kv_heads, self.d
        out = torch.zeros((self.rows, self.heads, d), dtype=torch.float64, device="cuda")
        lse = torch.full((self.rows, self.heads), -math.inf, dtype=torch.float64, device="cuda")
        tol, tol_l = torch.zeros_like(out), torch.zeros((self.rows, self.heads), dtype=torch.float64, device="cuda")
        for i, (n_q, n) in enumerate(self.lens):
            a = int(self.cu_np[i])
            if n_q == 0 or n == 0:
                continue
            at = torch.from_numpy(self.slots(i, n)).cuda()
            seen = torch.arange(n, device="cuda")[None] <= torch.arange(n_q, device="cuda")[:, None] + (n - n_q)
            for h in range(self.kv_heads):
                k, v = self.k[at, h].double() * self.k_scale, self.v[at, h].double() * self.v_scale
                for e in range(h * g, h * g + g):
                    q = self.q[a:a + n_q, e * d:(e + 1) * d].double()
                    s = torch.where(seen, q @ k.T * self.scale, -math.inf)
                    off = torch.where(seen, q.abs() @ k.abs().T * self.scale, 0.0).amax(-1, keepdim=True) * (d + 4) * 2.0 ** -23
                    top = s.amax(-1, keepdim=True)
                    ok = top > -math.inf
                    p = torch.where(seen & ok, torch.exp(s - torch.where(ok, top, 0.0)), 0.0)
                    total = p.sum(-1, keepdim=True)
                    err = 1.01 * off + 2.0 ** -21 + n * 2.0 ** -24
                    o = torch.where(ok, p @ v / total, 0.0)
                    mag = torch.where(ok, p @ v.abs() / total, 0.0)
                    step = 2.0 ** -11 if self.fp8 else 2.0 ** -8
                    small = torch.where(ok, seen.double() @ v.abs() / total, 0.0) * (2.0 ** -25 if self.fp8 else 0.0)
                    out[a:a + n_q, e] = o
                    tol[a:a + n_q, e] = mag * (2 * err + step + n * 2.0 ** -23) + small + o.abs() * 2.0 ** -8 + 1e-30
                    lse[a:a + n_q, e] = torch.where(ok, top + torch.log(total), -math.inf)[:, 0]
                    tol_l[a:a + n_q, e] = (2 * err + lse[a:a + n_q, e:e + 1].abs().clamp(max=1e30) * 2.0 ** -22 + 2.0 ** -22)[:, 0]
        return out, lse, tol, tol_l

    def check(self, lse=True):
        torch = self.torch
        torch.cuda.synchronize()
        out, want_l, tol, tol_l = self.exact()
        got = self.out[:self.rows].double().view(out.shape)
        assert torch.isfinite(got).all()
        over = (got - out).abs() - tol
        assert (over <= 0).all(), f"off by {(got - out).abs().max().item()}, {over.max().item()} over the bound at {np.unravel_index(int(over.argmax()), out.shape)}"
        assert (self.out[self.rows:] == 77.0).all()                       # rows behind the last sequence
        if lse:
            got = self.lse[:self.rows].double()
            none = torch.isinf(want_l)
            assert torch.equal(torch.isinf(got), none)
            assert ((got - want_l).abs()[~none] <= tol_l[~none]).all()
            assert (self.lse[self.rows:] == 77.0).all()
        assert self.atlas.device_status() == 0
