"""The operators around the paged K/V cache, as cases that can be timed: the attention that reads it, the decode-path writer
of an E4M3 cache, and what is done with its pages between two steps of a server.

A case is a dict of plain values with a "kind":

  attention  every sequence of a batch has a chunk of new tokens (one while it decodes, a few while drafts are verified, many
             while its prompt is read) whose keys and values stand in the paged cache already; each new token attends to all
             that stands before it and to itself.
  write      the QKV consumer of a decode step: per-head norm and rotation of Q (in place) and K, K and V into E4M3 pages.
  step       drafts of the last step are freed, every live sequence is forked into new ones (full pages shared, the last,
             part-filled one copied, over all layers), and each draft gets pages for some more tokens.
  compact    pages in use move down until they are the first of the pool, over all layers; tables follow.

Which sequence is how long is part of a case and goes by its numbers alone; pages, tokens and values go by the seed.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

EPS, THETA = 1e-6, 1e6
K_SCALE, V_SCALE = 0.03125, 0.015625          # what a code of the E4M3 caches stands for


def _ab():
    path = os.path.join(os.getcwd(), "apathy-atlas_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import atlas_b200
    return atlas_b200


def listed():
    return [
        # one user, one token: the smallest call, where latency is all there is
        dict(name="decode_1", kind="attention", seqs=1, q_len=1, kv_len=777, ragged=False, heads=32, kv_heads=8, head_dim=128,
             page=16, cache="bf16", lse=False),
        # a decode batch of sequences between a few tokens and 8192
        dict(name="decode_64", kind="attention", seqs=64, q_len=1, kv_len=8192, ragged=True, heads=32, kv_heads=8, head_dim=128,
             page=16, cache="bf16", lse=False),
        # a wide decode batch over an E4M3 cache
        dict(name="decode_fp8_256", kind="attention", seqs=256, q_len=1, kv_len=4096, ragged=True, heads=64, kv_heads=8, head_dim=128,
             page=32, cache="e4m3", lse=False),
        # a few prompts' chunks of odd lengths, small heads, pages that no power of two divides
        dict(name="chunk_odd_333", kind="attention", seqs=5, q_len=333, kv_len=2777, ragged=True, heads=24, kv_heads=8, head_dim=64,
             page=24, cache="bf16", lse=True),
        # one chunk of a chunked prefill deep into a long prompt, E4M3 cache
        dict(name="chunk_512_fp8_32k", kind="attention", seqs=1, q_len=512, kv_len=32768, ragged=False, heads=32, kv_heads=8, head_dim=128,
             page=64, cache="e4m3", lse=True),
        # the largest: a prompt of 8192 tokens at once
        dict(name="prefill_8192", kind="attention", seqs=1, q_len=8192, kv_len=8192, ragged=False, heads=32, kv_heads=8, head_dim=128,
             page=16, cache="bf16", lse=False),
        # the writer of a decode batch ...
        dict(name="write_fp8_64", kind="write", tokens=64, heads=32, kv_heads=8, head_dim=128, rotary=128, page=16),
        # ... and of a prefill batch
        dict(name="write_fp8_8192", kind="write", tokens=8192, heads=32, kv_heads=8, head_dim=128, rotary=64, page=16),
        # one user's drafts: two branches of five tokens
        dict(name="step_1x2", kind="step", live=1, drafts=2, new=5, kv_len=900, layers=8, kv_heads=8, head_dim=128, page=16, spare=64),
        # a server's: 48 sequences of four drafts each
        dict(name="step_48x4", kind="step", live=48, drafts=4, new=3, kv_len=2048, layers=8, kv_heads=8, head_dim=128, page=32, spare=512),
        # a small pool, half in use
        dict(name="compact_300", kind="compact", pages=300, seqs=7, used=0.5, layers=4, kv_heads=8, head_dim=128, page=16),
        # a large one, two thirds in use
        dict(name="compact_4000", kind="compact", pages=4000, seqs=80, used=0.66, layers=8, kv_heads=8, head_dim=128, page=16),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(("attention", "write", "step", "compact"), (6, 1.5, 1.5, 1))[0]
    page = rng.choice((5, 8, 16, 16, 24, 32, 64, 128, 256))
    kv_heads, head_dim = rng.choice((1, 2, 4, 8)), rng.choice((64, 96, 128, 128, 256))
    if kind == "attention":
        group = rng.choice((1, 2, 3, 4, 4, 7, 8, 16))
        form = rng.choice(("decode", "decode", "verify", "chunk", "chunk"))
        cache = rng.choice(("bf16", "bf16", "e4m3"))
        heads = kv_heads * group
        q_len = 1 if form == "decode" else rng.randint(2, 16) if form == "verify" else _log_int(rng, 17, 8192)
        seqs = _log_int(rng, 1, 256) if form != "chunk" else _log_int(rng, 1, 8)
        most = (1 << (30 if cache == "e4m3" else 29)) // (seqs * kv_heads * head_dim)       # values of the cache
        most = min(most, int((1 << 31) / (seqs * heads * q_len)), int(1.37e11 / (seqs * heads * q_len * head_dim)))
        while most < q_len:                                                                # no more work than the largest listed case
            seqs, q_len = max(1, seqs // 2), max(1, q_len // 2)
            most = int(min((1 << 29) / (seqs * kv_heads * head_dim), (1 << 31) / (seqs * heads * q_len), 1.37e11 / (seqs * heads * q_len * head_dim)))
        return dict(kind=kind, seqs=seqs, q_len=q_len, kv_len=_log_int(rng, q_len, max(q_len, min(131072, most))), ragged=seqs > 1 and rng.random() < 0.8,
                    heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page, cache=cache, lse=rng.random() < 0.3)
    if kind == "write":
        group = rng.choice((1, 2, 4, 8))
        most = 8192 * 40 * 128 // (kv_heads * (group + 2) * head_dim)
        return dict(kind=kind, tokens=_log_int(rng, 1, min(8192, most)), heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
                    rotary=rng.choice((64, head_dim)), page=page)
    if kind == "step":
        live, drafts = _log_int(rng, 1, 48), rng.randint(1, 4)
        return dict(kind=kind, live=live, drafts=drafts, new=rng.randint(1, 7), kv_len=_log_int(rng, 1, 2048), layers=rng.randint(1, 8), kv_heads=kv_heads,
                    head_dim=min(head_dim, 128), page=min(page, 32), spare=rng.randint(0, 300))
    return dict(kind=kind, pages=_log_int(rng, 30, 4000), seqs=_log_int(rng, 1, 60), used=round(rng.uniform(0.2, 0.9), 2), layers=rng.randint(1, 8),
                kv_heads=kv_heads, head_dim=min(head_dim, 128), page=min(page, 16))


# ---------------------------------------------------------------------------------------------------------------------
# lengths, which go by the case alone
# ---------------------------------------------------------------------------------------------------------------------
def _lens(case):
    """(new tokens, cached tokens) of every sequence of an attention case; a ragged batch has one without new tokens."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["q_len"], case["kv_len"]))
    lens = [(case["q_len"], case["kv_len"])]
    for i in range(1, case["seqs"]):
        q = rng.randint(max(1, case["q_len"] // 2), case["q_len"]) if case["ragged"] else case["q_len"]
        kv = rng.randint(q, case["kv_len"]) if case["ragged"] else case["kv_len"]
        lens.append((0 if case["ragged"] and i == 3 else q, kv))
    rng.shuffle(lens)
    return lens


def _live_lens(case):
    rng = random.Random("%d %d %d" % (case["live"], case["kv_len"], case["page"]))
    return [case["kv_len"]] + [rng.randint(1, case["kv_len"]) for _ in range(case["live"] - 1)]


def _pool_lens(case):
    """Sequences of a pool of which `used` of the pages are in use; the last one ends inside a page."""
    total = max(1, int(case["pages"] * case["used"]))
    seqs = min(case["seqs"], total)
    rng = random.Random("%d %d" % (case["pages"], seqs))
    cuts = [0] + sorted(rng.sample(range(1, total), seqs - 1)) + [total] if seqs > 1 else [0, total]
    lens = [(b - a) * case["page"] for a, b in zip(cuts, cuts[1:])]
    return [n - rng.randint(0, case["page"] - 1) for n in lens]


def _pages(n, page):
    return (n + page - 1) // page


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _normal(shape, g, dtype=torch.float32):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 27):
        part = flat[at:at + (1 << 27)]
        part.copy_(torch.randn(part.numel(), generator=g, device="cuda"))
    return out


def _codes(shape, g):
    """An E4M3 cache of values |N(0, 1)| / 16 or so: codes around 1."""
    out = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 27):
        part = flat[at:at + (1 << 27)]
        part.copy_(torch.randn(part.numel(), generator=g, device="cuda") / K_SCALE)
    return out


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    return {"attention": _prepare_attention, "write": _prepare_write, "step": _prepare_step, "compact": _prepare_compact}[case["kind"]](case, seed)


def _tables(lens, page, n_pages, stride, rng):
    """A page of the pool's own for every page of every sequence, in no order; -1 behind the last."""
    free = rng.permutation(n_pages)
    table = np.full((len(lens), stride), -1, np.int32)
    at = 0
    for i, n in enumerate(lens):
        k = _pages(n, page)
        table[i, :k] = free[at:at + k]
        at += k
    return table


def _prepare_attention(case, seed):
    g, rng = _gen(seed), np.random.default_rng(seed)
    lens, page, d = _lens(case), case["page"], case["head_dim"]
    used = sum(_pages(kv, page) for _, kv in lens)
    n_pages, stride = used + 3, _pages(case["kv_len"], page)
    shape = (n_pages, page, case["kv_heads"], d)
    make = _codes if case["cache"] == "e4m3" else lambda s, gen: _normal(s, gen, torch.bfloat16)
    s = dict(case, k_cache=make(shape, g), v_cache=make(shape, g))
    cu = np.concatenate([[0], np.cumsum([q for q, _ in lens])]).astype(np.int32)
    # heads differ in how sharply they look: standard deviations of the scores between 1 and 4
    sharp = torch.exp2(torch.linspace(0, 2, case["heads"], device="cuda")).view(1, -1, 1)
    s["q"] = (_normal((int(cu[-1]), case["heads"], d), g) * sharp).to(torch.bfloat16)
    s["table"] = torch.from_numpy(_tables([kv for _, kv in lens], page, n_pages, stride, rng)).cuda()
    s["cu_q"], s["kv_lens"] = torch.from_numpy(cu).cuda(), _i32([kv for _, kv in lens])
    s["scales"] = (K_SCALE, K_SCALE) if case["cache"] == "e4m3" else (1.0, 1.0)
    s["out"] = torch.empty_like(s["q"])
    s["lse_out"] = torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda") if case["lse"] else None
    if own:
        ab = _ab()
        desc = ab.make_attention_desc(
            q=s["q"], out=s["out"], lse=s["lse_out"], k_cache=s["k_cache"], v_cache=s["v_cache"], block_table=s["table"], cu_q=s["cu_q"],
            kv_len=s["kv_lens"], n_seqs=len(lens), n_tokens=int(cu[-1]), max_q_len=case["q_len"], max_kv_len=case["kv_len"], n_pages=n_pages,
            table_stride=stride, q_heads=case["heads"], kv_heads=case["kv_heads"], head_dim=d, block_size=page,
            softmax_scale=1.0 / math.sqrt(d), cache_dtype=ab.CACHE_E4M3 if case["cache"] == "e4m3" else ab.CACHE_BF16,
            k_scale=s["scales"][0], v_scale=s["scales"][1])
        s["ws"] = torch.zeros(ab.attention_ws_bytes(desc), dtype=torch.uint8, device="cuda")
        desc.ws, desc.ws_bytes = s["ws"].data_ptr(), s["ws"].numel()
        s["desc"] = desc
    return s


def _prepare_write(case, seed):
    g, rng = _gen(seed), np.random.default_rng(seed)
    t, hq, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    n_pages = _pages(t, case["page"]) + 2
    slots = rng.permutation(n_pages * case["page"])[:t].astype(np.int64)
    if t > 8:
        slots[rng.integers(0, t)] = -1                   # a padding token
    size = torch.exp2(torch.rand((t, 1), generator=g, device="cuda") * 6 - 3)
    freq = THETA ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64, device="cuda") / case["rotary"])
    qkv = _normal((t, (hq + 2 * hk) * d), g)
    qkv[:, :(hq + hk) * d] *= size
    return dict(case, qkv=qkv.to(torch.bfloat16),
                q_w=(0.1 * _normal((d,), g)).to(torch.bfloat16), k_w=(0.1 * _normal((d,), g)).to(torch.bfloat16),
                positions=torch.from_numpy(rng.integers(0, 131072, t).astype(np.int32)).cuda(), inv_freq=freq.float(),
                slots=torch.from_numpy(slots).cuda(),
                k_cache=torch.zeros((n_pages, case["page"], hk, d), dtype=torch.float8_e4m3fn, device="cuda"),
                v_cache=torch.zeros((n_pages, case["page"], hk, d), dtype=torch.float8_e4m3fn, device="cuda"))


def _pool(case, lens, n_pages, stride, more_seqs, seed):
    """K and V of all layers, [2 layers, pages, page, heads, width], and the tables of `lens` (and of `more_seqs` empty sequences)."""
    g, rng = _gen(seed), np.random.default_rng(seed)
    table = np.full((len(lens) + more_seqs, stride), -1, np.int32)
    table[:len(lens)] = _tables(lens, case["page"], n_pages, stride, rng)
    ref = np.zeros(n_pages, np.int32)
    ref[table[table >= 0]] = 1
    caches = _normal((2 * case["layers"], n_pages, case["page"], case["kv_heads"], case["head_dim"]), g, torch.bfloat16)
    s = dict(case, caches=caches, table=torch.from_numpy(table).cuda(), ref=torch.from_numpy(ref).cuda(), lens=_i32(list(lens) + [0] * more_seqs),
             bases=torch.tensor([c.data_ptr() for c in caches], dtype=torch.int64, device="cuda"))
    if own:
        ab = _ab()
        s["pages_desc"] = ab.make_cache_desc(
            bases=s["bases"], n_bases=2 * case["layers"], page_bytes=caches[0, 0].numel() * 2, n_pages=n_pages, block_size=case["page"],
            refcount=s["ref"], block_table=s["table"], table_stride=stride, seq_len=s["lens"], n_seqs=len(table))
        s["ws"] = torch.zeros(ab.cache_ws_bytes(s["pages_desc"], len(table)), dtype=torch.uint8, device="cuda")
        s["pages_desc"].ws, s["pages_desc"].ws_bytes = s["ws"].data_ptr(), s["ws"].numel()
    return s


def _prepare_step(case, seed):
    lens, page = _live_lens(case), case["page"]
    n = case["live"] * case["drafts"]
    each = _pages(page - 1 + case["new"], page)
    stride = _pages(case["kv_len"] + case["new"], page)
    s = _pool(case, lens, sum(_pages(k, page) for k in lens) + n * (each + 1) + case["spare"], stride, n, seed)
    # drafts go to parents in no order; each gets between one and `new` tokens
    rng = np.random.default_rng(seed)
    s["src"] = torch.from_numpy(rng.permutation(np.repeat(np.arange(case["live"]), case["drafts"])).astype(np.int32)).cuda()
    s["dst"] = torch.arange(case["live"], case["live"] + n, dtype=torch.int32, device="cuda")
    s["n_new"] = torch.from_numpy(rng.integers(1, case["new"] + 1, n).astype(np.int32)).cuda()
    s["slots"] = torch.empty(n * case["new"], dtype=torch.int64, device="cuda")
    s["fork_status"], s["append_status"] = (torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(2))
    return s


def _prepare_compact(case, seed):
    lens = _pool_lens(case)
    s = _pool(case, lens, case["pages"], max(_pages(k, case["page"]) for k in lens), 0, seed)
    s["ref_out"], s["table_out"] = torch.empty_like(s["ref"]), torch.empty_like(s["table"])
    s["map"], s["n_used"] = torch.empty_like(s["ref"]), torch.empty(1, dtype=torch.int32, device="cuda")
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    return {"attention": _run_attention, "write": _run_write, "step": _run_step, "compact": _run_compact}[state["kind"]](state)


def _run_attention(s):
    if own:
        _ab().paged_attention(s["desc"])
        return [s["out"], s["lse_out"]] if s["lse"] else [s["out"]]
    seqs, q_max, kv_max, page = s["seqs"], s["q_len"], s["kv_len"], s["page"]
    hk, d = s["kv_heads"], s["head_dim"]
    g = s["heads"] // hk
    cu, kv = s["cu_q"].long(), s["kv_lens"].long()
    j = torch.arange(kv_max, device="cuda")
    inside = j < kv[:, None]                                                                   # [seqs, kv_max]
    row = torch.where(inside, s["table"].long()[:, j // page] * page + j % page, 0)
    k = s["k_cache"].flatten(0, 1)[row].float() * s["scales"][0]                              # [seqs, kv_max, hk, d]
    v = torch.where(inside[..., None, None], s["v_cache"].flatten(0, 1)[row].float() * s["scales"][1], 0.0)
    i = torch.arange(q_max, device="cuda")
    q_len = cu[1:] - cu[:-1]
    there = i < q_len[:, None]                                                                # [seqs, q_max]
    token = torch.where(there, cu[:-1, None] + i, 0)
    q = s["q"][token].float().view(seqs, q_max, hk, g, d).permute(0, 2, 3, 1, 4).reshape(seqs, hk, g * q_max, d)
    score = (q @ k.permute(0, 2, 3, 1)).view(seqs, hk, g, q_max, kv_max) * (1.0 / math.sqrt(d))
    last = (kv - q_len)[:, None] + i                                                          # the last position a row sees
    seen = inside[:, None, :] & (j <= last[..., None]) & there[..., None]                     # [seqs, q_max, kv_max]
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = (p.view(seqs, hk, g * q_max, kv_max) @ v.permute(0, 2, 1, 3)).view(seqs, hk, g, q_max, d)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(seqs, q_max, s["heads"], d)
    s["out"][token[there]] = out[there].to(torch.bfloat16)
    if not s["lse"]:
        return [s["out"]]
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2).reshape(seqs, q_max, s["heads"])
    s["lse_out"][token[there]] = lse[there]
    return [s["out"], s["lse_out"]]


def _run_write(s):
    t, hq, hk, d, rot = s["tokens"], s["heads"], s["kv_heads"], s["head_dim"], s["rotary"]
    qw, kw = hq * d, hk * d
    if own:
        base, stride = s["qkv"].data_ptr(), qw + 2 * kw
        _ab().qkv_norm_rope_cache_write_fp8(base, base + 2 * qw, base + 2 * (qw + kw), stride, stride, s["q_w"], s["k_w"], s["positions"], s["inv_freq"],
                                            s["slots"], s["k_cache"], s["v_cache"], t, hq, hk, d, rot, s["page"], EPS, 1.0 / K_SCALE, 1.0 / V_SCALE)
        return [s["qkv"], s["k_cache"], s["v_cache"]]
    x = s["qkv"].view(t, hq + 2 * hk, d)
    qk = x[:, :hq + hk].float()
    w = torch.cat([s["q_w"].float().expand(hq, d), s["k_w"].float().expand(hk, d)]) + 1.0
    qk = (qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS) * w).to(torch.bfloat16).float()
    # the angle is the FP32 product of position and frequency; its cosine and sine in 64 bits, because it is far beyond a turn
    angle = (s["positions"].float()[:, None] * s["inv_freq"]).double()[:, None, :]
    c, sn = torch.cos(angle).float(), torch.sin(angle).float()
    a, b = qk[..., :rot // 2], qk[..., rot // 2:rot]
    y = torch.cat([a * c - b * sn, b * c + a * sn, qk[..., rot:]], -1)
    x[:, :hq] = y[:, :hq].to(torch.bfloat16)
    live = s["slots"] >= 0
    at = s["slots"][live]
    s["k_cache"].flatten(0, 1)[at] = (y[:, hq:] * (1.0 / K_SCALE)).clamp(-448, 448).to(torch.float8_e4m3fn)[live]
    s["v_cache"].flatten(0, 1)[at] = (x[:, hq + hk:].float() * (1.0 / V_SCALE)).clamp(-448, 448).to(torch.float8_e4m3fn)[live]
    return [s["qkv"], s["k_cache"], s["v_cache"]]


def _nth_free(ref, n):
    """The first n pages that nothing refers to, in order (a page behind the pool where there are fewer), and how many there are."""
    count = torch.cumsum((ref == 0).long(), 0)
    return torch.searchsorted(count, torch.arange(1, n + 1, device="cuda")), count[-1]


def _run_step(s):
    n = s["src"].numel()
    outs = [s["fork_status"], s["append_status"], s["slots"], s["lens"], s["table"], s["ref"], s["caches"]]
    if own:
        ab, desc = _ab(), s["pages_desc"]
        ab.cache_free(desc, s["dst"], n)
        ab.cache_fork(desc, s["src"], s["dst"], n, s["fork_status"])
        ab.cache_append(desc, s["dst"], s["n_new"], n, s["slots"], s["slots"].numel(), s["append_status"])
        return outs
    page, table, ref, lens = s["page"], s["table"], s["ref"], s["lens"]
    src, dst, stride = s["src"].long(), s["dst"].long(), table.shape[1]
    cols = torch.arange(stride, device="cuda")
    # free
    held = cols < ((lens[dst].long() + page - 1) // page)[:, None]
    ref.index_add_(0, table[dst].clamp(min=0).long().view(-1), -held.int().view(-1))
    table[dst] = torch.where(held, -1, table[dst])
    lens[dst] = 0
    # fork
    size = lens[src].long()
    full, rest = size // page, size % page
    need = (rest > 0).long()
    before = torch.cumsum(need, 0) - need
    free, there = _nth_free(ref, n)
    ok = (need == 0) | (before + need <= there)
    shared = (cols < full[:, None]) & ok[:, None]
    ref.index_add_(0, table[src].clamp(min=0).long().view(-1), shared.int().view(-1))
    part = (need > 0) & ok
    fresh = free[before[part]]
    old = table[src[part], full[part]].long()
    ref[fresh] = 1
    row = torch.where(shared, table[src], -1)
    row[part, full[part]] = fresh.int()
    table[dst] = row
    lens[dst] = torch.where(ok, size, 0).int()
    used = (torch.arange(page, device="cuda") < rest[part][:, None])[None, ..., None, None]
    s["caches"][:, fresh] = torch.where(used, s["caches"][:, old], s["caches"][:, fresh])
    s["fork_status"].copy_(torch.where(ok, 0, -5))
    # append
    new = s["n_new"].long()
    size = lens[dst].long()
    have, want = (size + page - 1) // page, (size + new + page - 1) // page
    need = want - have
    before = torch.cumsum(need, 0) - need
    free, there = _nth_free(ref, n * (_pages(s["new"], page) + 1))
    ok = ((need == 0) | (before + need <= there)) & (want <= stride)
    put = (cols >= have[:, None]) & (cols < want[:, None]) & ok[:, None]
    fresh = free[(before[:, None] + cols - have[:, None])[put]]
    ref[fresh] = 1
    row = table[dst]
    row[put] = fresh.int()
    table[dst] = row
    lens[dst] = torch.where(ok, size + new, size).int()
    k = torch.arange(s["new"], device="cuda")
    mine = k < new[:, None]
    at = size[:, None] + k
    slot = torch.gather(row.long(), 1, (at // page).clamp(max=stride - 1)) * page + at % page
    first = torch.cumsum(new, 0) - new
    s["slots"].fill_(-1)
    s["slots"][(first[:, None] + k)[mine]] = torch.where(ok[:, None], slot, -1)[mine]
    s["append_status"].copy_(torch.where(ok, 0, -5))
    return outs


def _run_compact(s):
    outs = [s["n_used"], s["map"], s["ref_out"], s["table_out"], s["caches"]]
    if own:
        _ab().cache_compact(s["pages_desc"], s["ref_out"], s["table_out"], s["map"], s["n_used"])
        return outs
    n_pages = s["ref"].numel()
    used = s["ref"] > 0
    u = used.sum()
    idx = torch.arange(n_pages, device="cuda")
    movers, holes = torch.nonzero(used & (idx >= u)).view(-1), torch.nonzero(~used & (idx < u)).view(-1)
    s["map"].copy_(torch.where(used, idx, -1))
    s["map"][movers] = holes.int()
    s["n_used"].copy_(u)
    s["ref_out"].copy_(torch.where(idx < u, s["ref"], 0))
    s["ref_out"][holes] = s["ref"][movers]
    held = torch.arange(s["table"].shape[1], device="cuda") < ((s["lens"].long() + s["page"] - 1) // s["page"])[:, None]
    s["table_out"].copy_(torch.where(held, s["map"][s["table"].long().clamp(min=0)], s["table"]))
    s["caches"][:, holes] = s["caches"][:, movers]
    return outs


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    kind, page = case["kind"], case.get("page")
    if kind == "attention":
        lens, d = _lens(case), case["head_dim"]
        pairs = sum(q * kv - q * (q - 1) // 2 for q, kv in lens)
        tokens, size = sum(q for q, _ in lens), 1 if case["cache"] == "e4m3" else 2
        cached = sum(kv for q, kv in lens if q)
        return {"bytes": cached * case["kv_heads"] * d * 2 * size + tokens * case["heads"] * (4 * d + 4 * case["lse"]) + 4 * sum(_pages(kv, page) for q, kv in lens if q),
                "flops": 4 * pairs * case["heads"] * d}
    if kind == "write":
        t, d = case["tokens"], case["head_dim"]
        return {"bytes": t * d * (case["heads"] * 4 + case["kv_heads"] * 2 * 3) + 12 * t, "flops": t * (case["heads"] + case["kv_heads"]) * d * 8}
    token = case["kv_heads"] * case["head_dim"] * 2 * 2 * case["layers"]
    if kind == "step":
        lens = _live_lens(case)
        n = case["live"] * case["drafts"]
        return {"bytes": case["drafts"] * sum(k % page for k in lens) * token * 2 + 4 * 4 * case["drafts"] * sum(_pages(k, page) for k in lens) + 60 * n, "flops": 0}
    # pages in use stand anywhere: of U, a share U / pages stands among the first U already
    total = sum(_pages(k, page) for k in _pool_lens(case))
    return {"bytes": total * (1 - total / case["pages"]) * page * token * 2 + 12 * case["pages"] + 8 * total, "flops": 0}


# ---------------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits and one sequence at a time
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(s)
    if case["kind"] == "write":
        return _exact_write(s)
    return None                                           # whole numbers and copies


def _exact_attention(s):
    g, d, page = s["heads"] // s["kv_heads"], s["head_dim"], s["page"]
    cu, kv_lens, table = s["cu_q"].tolist(), s["kv_lens"].tolist(), s["table"].long()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for i, n in enumerate(kv_lens):
        a, b = cu[i], cu[i + 1]
        if a == b:
            continue
        pages = table[i, :_pages(n, page)]
        place = torch.arange(b - a, device="cuda") + n - (b - a)
        hidden = torch.arange(n, device="cuda") > place[:, None]
        for h in range(s["kv_heads"]):
            k = s["k_cache"][pages, :, h].reshape(-1, d)[:n].double() * s["scales"][0]
            v = s["v_cache"][pages, :, h].reshape(-1, d)[:n].double() * s["scales"][1]
            for e in range(h * g, h * g + g):
                score = (s["q"][a:b, e].double() @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf)
                lse[a:b, e] = torch.logsumexp(score, -1)
                out[a:b, e] = torch.softmax(score, -1) @ v
    return [out, lse] if s["lse"] else [out]


def _exact_write(s):
    hq, hk, d, half = s["heads"], s["kv_heads"], s["head_dim"], s["rotary"] // 2
    x = s["qkv"].double().view(s["tokens"], -1, d)
    result, k_rows = x.clone(), torch.empty_like(x[:, :hk])
    # the angle as the operator defines it: the FP32 product
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), (s["positions"].float()[:, None] * s["inv_freq"]).double())
    for h in range(hq + hk):
        w = (s["q_w"] if h < hq else s["k_w"]).double() + 1.0
        r = x[:, h]
        r = r / torch.sqrt((r * r).sum(-1, keepdim=True) / d + EPS) * w
        r = r.to(torch.bfloat16).double()                 # the operator rounds the normed head
        z = torch.complex(r[:, :half], r[:, half:2 * half]) * turn
        r[:, :half], r[:, half:2 * half] = z.real, z.imag
        if h < hq:
            result[:, h] = r
        else:
            k_rows[:, h - hq] = r
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    for t, slot in enumerate(s["slots"].tolist()):
        if slot >= 0:
            k_cache[slot // s["page"], slot % s["page"]] = (k_rows[t] / K_SCALE).clip(-448, 448)
            v_cache[slot // s["page"], slot % s["page"]] = (x[t, hq + hk:] / V_SCALE).clip(-448, 448)
    return [result.view(s["tokens"], -1), k_cache, v_cache]
