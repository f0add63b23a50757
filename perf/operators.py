"""Cases for the operators of serving several continuations from a 4-bit paged KV cache.

  decode    one-token GQA attention over a cache held in 4 bits (with or
            without the new token's fused append, RoPE, window, softcap)
  append    K/V rows quantised to 4 bits into the pages and read back
  pages     page lists copied inside a cache (copy on write after a fork,
            compaction)
  logprobs  log probabilities of given tokens, entropy and top alternatives
            over rows of logits

A 4-bit cache is held as blocks of 16 tokens of one kv head, 1024 bytes of
codes and 128 bytes of f16 scales each, pools [pages, kv heads, page / 16,
1152].  Every group of 32 dims of a row has a scale s = f16(max|x| / 7); a
value is (n - 8) s with n = clamp(rint(x / s), -7, 7) + 8.  In a K block the
32-bit word [token][t][group] holds dims 32 group + 8 t + {0, 2, 4, 6} in the
nibbles of its low half and the odd ones in its high half; in a V block the
16-bit half [token >> 3][g][(token >> 1) & 3][group][token & 1] holds dims
32 group + 4 g + {0, 1, 2, 3}.  K scales are [token][group], V scales
[token >> 1][group][token & 1].
"""
import math

import numpy as np
import torch

own = False

D, GROUPS, BLOCK, CODES, BLOCK_BYTES = 128, 4, 16, 1024, 1152
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- cases -----------------------------------------------------------------
def listed():
    return [
        # an interactive request: one sequence, a short context, the next token appended and attended
        _decode("decode 1 x 100", 1, 100, 100, append=True, rope=True),
        # the serving batch of the f16 benchmark: 64 sequences, ragged contexts
        _decode("decode 64 x 1k-8k", 64, 1024, 8192),
        # the int8 benchmark's long contexts, a whole step's attention with append and RoPE
        _decode("decode 32 x 8k-32k", 32, 8192, 32768, append=True, rope=True),
        # one very long document, odd length, few kv heads, larger pages: the work has to be split along it
        _decode("decode 1 x 130001", 1, 130001, 130001, heads=16, kv_heads=2, page=64),
        # sliding-window layers with a score cap and an odd head group; some sequences still empty
        _decode("decode 48 window", 48, 0, 6000, heads=20, kv_heads=4, page=32, window=1024, softcap=50.0),
        # one decode step's rows, as a separate write
        _append("append 32 x 1", 32, 1, 0, 4096, rope=True),
        # chunked prompts of the int8 append benchmark
        _append("append 32 x 512", 32, 512, 0, 4096),
        # one odd-sized prompt at an odd place in its page, few kv heads
        _append("append 1 x 8191", 1, 8191, 5, 5, kv_heads=2, rope=True),
        # copy on write: the shared last page of eight continuations, 4-bit pool
        _pages("pages fork 8", "int4", 256, 8),
        # compaction of half of a large f16 pool
        _pages("pages move 8000", "f16", 16384, 8000),
        # one sampled token with its alternatives
        _logprobs("logprobs 1 x 32000", 1, 32000, "f32", 5),
        # a decode batch with a grammar's mask, odd vocabulary
        _logprobs("logprobs 64 x 128257", 64, 128257, "bf16", 20, masked=True),
    ]


def _decode(name, batch, lo, hi, heads=32, kv_heads=8, page=16, append=False, rope=False, window=0, softcap=0.0):
    c = {"op": "decode", "batch": batch, "lo": lo, "hi": hi, "heads": heads, "kv_heads": kv_heads, "page": page,
         "append": append, "rope": rope, "window": window, "softcap": softcap}
    return dict(c, name=name) if name else c


def _append(name, batch, tokens, lo, hi, kv_heads=8, page=16, rope=False):
    c = {"op": "append", "batch": batch, "tokens": tokens, "lo": lo, "hi": hi, "kv_heads": kv_heads, "page": page,
         "rope": rope}
    return dict(c, name=name) if name else c


def _pages(name, kv, pool, copies, kv_heads=8, page=16):
    c = {"op": "pages", "kv": kv, "pool": pool, "copies": copies, "kv_heads": kv_heads, "page": page}
    return dict(c, name=name) if name else c


def _logprobs(name, rows, vocab, dtype, top, masked=False):
    c = {"op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top, "masked": masked}
    return dict(c, name=name) if name else c


def _between(rng, lo, hi):
    """A whole number of [lo, hi], evenly over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "append", "pages", "logprobs"])
    if op == "decode":
        kv_heads = rng.choice([1, 2, 4, 8])
        batch = _between(rng, 1, 64)
        hi = _between(rng, 1, min(131072, 640000 * 8 // (kv_heads * batch)))
        window = rng.choice([0, 0, _between(rng, 1, 4096)])
        # windows and softcaps come with the layers that have them; the append needs a token to write
        return _decode(None, batch, rng.choice([1, hi, max(1, hi // 4)]), hi, kv_heads * rng.randint(1, 8), kv_heads,
                       rng.choice([16, 32, 64, 128]), rng.random() < 0.5, rng.random() < 0.5, window,
                       rng.choice([0.0, 0.0, 30.0]))
    if op == "append":
        kv_heads = rng.choice([1, 2, 4, 8])
        batch = _between(rng, 1, 64)
        tokens = _between(rng, 1, max(1, 130000 // (kv_heads * batch)))
        hi = rng.randint(0, 9000)
        return _append(None, batch, tokens, rng.choice([0, hi]), hi, kv_heads, rng.choice([16, 32, 64]),
                       rng.random() < 0.5)
    if op == "pages":
        pool = _between(rng, 64, 16384)
        return _pages(None, rng.choice(["f16", "int4"]), pool, _between(rng, 1, min(pool // 2, 8000)),
                      rng.choice([1, 2, 4, 8]), 16)
    rows = _between(rng, 1, 128)
    return _logprobs(None, rows, _between(rng, 1000, 140000), rng.choice(["f32", "f16", "bf16"]), rng.randint(0, 32),
                     rng.random() < 0.5)


def _lengths(case):
    """The case's lengths, evenly from lo to hi."""
    return np.round(np.linspace(case["lo"], case["hi"], case["batch"])).astype(np.int64)


def work(case):
    op = case["op"]
    if op == "decode":
        n = _lengths(case)
        seen = np.minimum(n, case["window"]) if case["window"] else n
        b, h, g = case["batch"], case["heads"], case["kv_heads"]
        pages = int((-(-seen // case["page"])).sum())
        kv = int(seen.sum()) * g * 2 * (D // 2 + 2 * GROUPS)
        more = b * g * (2 * D * 2 + 2 * (2 * D + 72)) if case["append"] else 0  # new rows in, 4-bit out, read back as f16
        return {"bytes": kv + b * h * D * (2 + 2) + 4 * (pages + b) + more, "flops": 4 * h * D * int(seen.sum())}
    if op == "append":
        rows = case["batch"] * case["tokens"] * case["kv_heads"] * 2
        return {"bytes": rows * (2 * D + 72 + 72 + 2 * D), "flops": rows * D * 6}
    if op == "pages":
        page = case["page"] * case["kv_heads"] * 2 * (2 * D if case["kv"] == "f16" else 72)
        back = case["copies"] * case["page"] * case["kv_heads"] * 2 * (72 + 2 * D) if case["kv"] == "int4" else 0
        return {"bytes": 2 * case["copies"] * page + back, "flops": 0}
    size = torch.empty((), dtype=TYPES[case["dtype"]]).element_size()
    return {"bytes": case["rows"] * (case["vocab"] * size + 4 + 8 + 8 * case["top"]),
            "flops": case["rows"] * case["vocab"] * 6}


# ---- inputs ----------------------------------------------------------------
def _rows(gen, shape):
    """f16 K or V rows: normal values, each dim with a strength of its own, as projections give them."""
    strength = 0.25 + 1.5 * torch.rand((D,), generator=gen, device="cuda")
    return (torch.randn(shape + (D,), generator=gen, device="cuda") * strength).half()


def _scales_and_codes(x):
    """x [..., 128] f32 -> f16 scales [..., 4] and codes 1..15 [..., 4, 32]."""
    x = x.reshape(x.shape[:-1] + (GROUPS, D // GROUPS))
    s = (x.abs().amax(-1) / 7.0).half()
    q = torch.round(x / s.float().clamp_min(1e-30).unsqueeze(-1)).clamp(-7, 7)
    return s, torch.where(s.unsqueeze(-1) > 0, q, torch.zeros_like(q)) + 8


def _blocks(x, is_v):
    """x [n, 16, 128] f16 -> [n, 1152] bytes of K or V blocks."""
    s, c = _scales_and_codes(x.float())
    n = x.shape[0]
    c = c.to(torch.uint8)
    if is_v:  # tokens [half, t, parity], dims [group, g, s]
        c = c.reshape(n, 2, 4, 2, GROUPS, 8, 4).permute(0, 1, 5, 2, 4, 3, 6)
        s = s.reshape(n, 8, 2, GROUPS).permute(0, 1, 3, 2)
    else:  # tokens, dims [group, t, pair, odd]
        c = c.reshape(n, 16, GROUPS, 4, 4, 2).permute(0, 1, 3, 2, 5, 4)
    c = c.reshape(n, CODES, 2)
    s = s.reshape(n, 64).contiguous().view(torch.uint8)
    return torch.cat([c[..., 0] | (c[..., 1] << 4), s], 1)


def _pool(gen, pages, kv_heads, page):
    """A filled 4-bit pool pair [pages, kv heads, page / 16, 1152]."""
    n, step, pools = pages * kv_heads * (page // BLOCK), 1 << 17, []
    for is_v in (False, True):
        pool = torch.empty((n, BLOCK_BYTES), dtype=torch.uint8, device="cuda")
        for at in range(0, n, step):
            pool[at:at + step] = _blocks(_rows(gen, (min(step, n - at), BLOCK)), is_v)
        pools.append(pool.view(pages, kv_heads, page // BLOCK, BLOCK_BYTES))
    return pools


def _table(gen, lengths, page):
    """A random block table for these lengths: [batch, widest] int32, -1 unmapped, and its number of pages."""
    need = torch.from_numpy(-(-lengths // page)).cuda()
    wide, count = max(1, int(need.max())), max(1, int(need.sum()))
    live = torch.arange(wide, device="cuda") < need[:, None]
    table = torch.full(live.shape, -1, dtype=torch.int32, device="cuda")
    table[live] = torch.randperm(count, generator=gen, device="cuda")[:int(need.sum())].int()
    return table, count


def _rope_table(positions):
    """[positions, 64, {cos, sin}] f32."""
    inv = 500000.0 ** (-np.arange(0, D, 2) / D)
    angle = np.arange(positions)[:, None] * inv
    return torch.from_numpy(np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    st = dict(case)
    op = case["op"]
    if op == "logprobs":
        r, v, dt = case["rows"], case["vocab"], TYPES[case["dtype"]]
        x = torch.randn((r, v), generator=gen, device="cuda") * 3.0
        if case["masked"]:  # a grammar forbids most tokens; at the last row it has nothing left
            x = x.masked_fill(torch.rand((r, v), generator=gen, device="cuda") < 0.8, -math.inf)
            x[1:][-1:] = -math.inf
        return st | {"logits": x.to(dt),
                     "tokens": torch.randint(0, v, (r,), generator=gen, device="cuda", dtype=torch.int32)}
    g, page = case["kv_heads"], case["page"]
    if op == "pages":
        n = case["pool"]
        if case["kv"] == "f16":
            st["k_pool"], st["v_pool"] = (_rows(gen, (n * page, g)) for _ in range(2))
        else:
            st["k_pool"], st["v_pool"] = _pool(gen, n, g, page)
        order = torch.randperm(n, generator=gen, device="cuda")[:2 * case["copies"]].cpu()
        # pairs (from, to), as the host's page pool hands them out
        st["pairs"] = order.view(2, -1).t().contiguous().int().numpy()
        # the continuations' tables: each one's copied page
        st["table"] = order[case["copies"]:].int().view(-1, 1).cuda()
        st["from"], st["to"] = order[:case["copies"]].cuda(), order[case["copies"]:].cuda()
        st["starts"] = torch.zeros(case["copies"], dtype=torch.int32, device="cuda")
        return st
    b = case["batch"]
    n = _lengths(case)[np.random.default_rng(seed).permutation(b)]
    if op == "append":
        st["table"], pages = _table(gen, n + case["tokens"], page)
        st["k_pool"], st["v_pool"] = (torch.zeros((pages, g, page // BLOCK, BLOCK_BYTES), dtype=torch.uint8,
                                                  device="cuda") for _ in range(2))
        st["new_k"], st["new_v"] = (_rows(gen, (b, case["tokens"], g)) for _ in range(2))
        st["starts"] = torch.from_numpy(n.astype(np.int32)).cuda()
        st["rope_table"] = _rope_table(int(n.max()) + case["tokens"]) if case["rope"] else None
        return st
    st["table"], pages = _table(gen, n, page)
    st["k_pool"], st["v_pool"] = _pool(gen, pages, g, page)
    st["q"] = torch.randn((b, case["heads"], D), generator=gen, device="cuda").half()
    st["lengths"] = torch.from_numpy(n.astype(np.int32)).cuda()
    st["new_k"], st["new_v"] = (_rows(gen, (b, g)) for _ in range(2))
    st["starts"] = torch.from_numpy(np.maximum(n - 1, 0).astype(np.int32)).cuda()
    st["rope_table"] = _rope_table(int(n.max()) + 1) if case["rope"] else None
    return st


# ---- one pass --------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _cache(st, kv_dtype):
    from doe_b200.kv import PagedKVCache

    return PagedKVCache.from_pools(st["k_pool"], st["v_pool"], page_size=st["page"], num_kv_heads=st["kv_heads"],
                                   head_dim=D, block_table=st["table"], kv_dtype=kv_dtype)


def _run_own(st):
    from doe_b200 import ops

    op = st["op"]
    if op == "logprobs":
        r = ops.token_logprobs(st["logits"], st["tokens"], top_k=st["top"])
        return {"logprob": r.logprob, "entropy": r.entropy, "ids": r.top_ids, "top": r.top_logprobs}
    if op == "pages":
        cache = _cache(st, st["kv"])
        ops.paged_copy_pages(cache, st["pairs"])
        if st["kv"] == "f16":
            return {"k": st["k_pool"], "v": st["v_pool"]}
        k, v = ops.paged_read(cache, st["starts"], st["page"])
        return {"k": k, "v": v}
    cache = _cache(st, "int4")
    if op == "append":
        ops.paged_append(cache, st["new_k"], st["new_v"], st["starts"], freq_cis=st["rope_table"])
        k, v = ops.paged_read(cache, st["starts"], st["tokens"])
        return {"k": k, "v": v}
    out = ops.paged_decode(cache, st["q"], st["lengths"], 1.0 / math.sqrt(D),
                           new_k=st["new_k"] if st["append"] else None, new_v=st["new_v"] if st["append"] else None,
                           freq_cis=st["rope_table"], sliding_window=st["window"], softcap=st["softcap"],
                           out_dtype=torch.bfloat16)
    if not st["append"]:
        return {"out": out}
    k, v = ops.paged_read(cache, st["starts"], 1)
    return {"out": out, "k": k, "v": v}


# ---- the plain form: elementary operations in 32 bits ------------------------
def _values(blocks, is_v):
    """[..., 1152] bytes -> [..., 16, 128] f32 values."""
    lead = blocks.shape[:-1]
    b = blocks[..., :CODES]
    c = torch.stack([b & 15, b >> 4], -1)
    s = blocks[..., CODES:].contiguous().view(torch.float16)
    k = len(lead)
    if is_v:
        c = c.view(lead + (2, 8, 4, GROUPS, 2, 4)).permute(tuple(range(k)) + (k, k + 2, k + 4, k + 3, k + 1, k + 5))
        s = s.view(lead + (8, GROUPS, 2)).transpose(-1, -2)
    else:
        c = c.view(lead + (16, 4, GROUPS, 2, 4)).permute(tuple(range(k)) + (k, k + 2, k + 1, k + 4, k + 3))
    c = c.reshape(lead + (16, GROUPS, 32)).float() - 8.0
    return (c * s.reshape(lead + (16, GROUPS, 1)).float()).view(lead + (16, D))


def _tokens(pool, table, is_v):
    """Every mapped token of the tables: [batch, kv heads, tokens, 128] f32."""
    x = _values(pool[table.clamp_min(0).long()], is_v)  # [batch, pages, kv heads, page / 16, 16, 128]
    return x.transpose(1, 2).reshape(x.shape[0], x.shape[2], -1, D)


def _rotate(x, at, rope_table):
    """x [..., heads, 128] f16 rotated at positions `at` [...], rounded to f16."""
    cis = rope_table[at.long()].unsqueeze(-3)
    c, s = cis[..., 0], cis[..., 1]
    x0, x1 = x.float().chunk(2, -1)
    return torch.cat([x0 * c - x1 * s, x0 * s + x1 * c], -1).half()


def _held(x):
    """f16 rows as a 4-bit cache holds them, f32."""
    s, c = _scales_and_codes(x.float())
    return ((c - 8) * s.float().unsqueeze(-1)).reshape(x.shape)


def _run_plain(st):
    op = st["op"]
    if op == "logprobs":
        x = st["logits"].float()
        m = x.amax(-1, keepdim=True)
        d = x - torch.where(m > -math.inf, m, torch.zeros_like(m))
        e = torch.exp(d)
        s = e.sum(-1)
        none = s == 0  # every token forbidden
        ls = torch.log(s)
        # a forbidden token adds nothing to the entropy
        h = ls - torch.where(e > 0, e * d, torch.zeros_like(e)).sum(-1) / s
        at = torch.gather(d, 1, st["tokens"].long()[:, None])[:, 0]
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :st["top"]]
        top = torch.gather(d, 1, ids)
        low = torch.full_like(s, -math.inf)
        return {"logprob": torch.where(none, low, at - ls), "entropy": torch.where(none, torch.zeros_like(h), h),
                "ids": ids.int(), "top": torch.where(none[:, None], low[:, None], top - ls[:, None])}
    if op == "pages":
        if st["kv"] == "f16":
            for pool in (st["k_pool"], st["v_pool"]):
                by_page = pool.view((st["pool"], st["page"]) + pool.shape[1:])
                by_page[st["to"]] = by_page[st["from"]]
            return {"k": st["k_pool"], "v": st["v_pool"]}
        for pool in (st["k_pool"], st["v_pool"]):
            pool[st["to"]] = pool[st["from"]]
        k, v = (_tokens(st[p], st["table"], p == "v_pool").transpose(1, 2).half() for p in ("k_pool", "v_pool"))
        return {"k": k, "v": v}
    if op == "append":
        k, v = st["new_k"], st["new_v"]
        if st["rope"]:
            at = st["starts"][:, None] + torch.arange(st["tokens"], device="cuda")
            k = _rotate(k, at, st["rope_table"])
        return {"k": _held(k).half(), "v": _held(v).half()}
    b, h, g = st["batch"], st["heads"], st["kv_heads"]
    n, q = st["lengths"], st["q"]
    if st["rope"]:
        q = _rotate(q, st["starts"], st["rope_table"])
    k, v = _tokens(st["k_pool"], st["table"], False), _tokens(st["v_pool"], st["table"], True)
    back = {}
    if st["append"]:
        nk = _rotate(st["new_k"], st["starts"], st["rope_table"]) if st["rope"] else st["new_k"]
        nk, nv = _held(nk), _held(st["new_v"])
        rows = torch.arange(b, device="cuda")
        k[rows, :, st["starts"].long()] = nk
        v[rows, :, st["starts"].long()] = nv
        back = {"k": nk.half()[:, None], "v": nv.half()[:, None]}
    x = (q.view(b, g, h // g, D).float() @ k.transpose(-1, -2)) / math.sqrt(D)  # [batch, kv heads, group, tokens]
    if st["softcap"]:
        x = st["softcap"] * torch.tanh(x / st["softcap"])
    at = torch.arange(k.shape[2], device="cuda")
    seen = at < n[:, None]
    if st["window"]:
        seen = seen & (at >= n[:, None] - st["window"])
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
    out = (e @ v) / e.sum(-1, keepdim=True).clamp_min(1e-30)
    return {"out": out.reshape(b, h, D).bfloat16()} | back


# ---- the definition in 64 bits ------------------------------------------------
def _place(is_v):
    """[16 tokens, 128 dims] -> the byte and the nibble that hold the code, and the half that holds the scale."""
    tok, dim = np.meshgrid(np.arange(16), np.arange(D), indexing="ij")
    group, d = dim // 32, dim % 32
    if is_v:
        half = (((tok // 8 * 8 + d // 4) * 4 + tok // 2 % 4) * GROUPS + group) * 2 + tok % 2
        byte, nibble = half * 2 + d % 4 // 2, d % 2
        scale = (tok // 2 * GROUPS + group) * 2 + tok % 2
    else:
        word = (tok * 4 + d // 8) * GROUPS + group
        slot = d % 8 // 2 + 4 * (d % 2)
        byte, nibble = word * 4 + slot // 2, slot % 2
        scale = tok * GROUPS + group
    return (torch.from_numpy(a).cuda() for a in (byte, nibble, scale))


def _exact_rows(blocks, is_v):
    byte, nibble, scale = _place(is_v)
    code = (blocks[..., byte].long() >> (4 * nibble)) & 15
    s = blocks[..., CODES:].contiguous().view(torch.float16).double()
    return (code - 8).double() * s[..., scale]


def _exact_held(x):
    x = x.cpu().double().numpy().reshape(x.shape[:-1] + (GROUPS, 32))
    s = (np.abs(x).max(-1, keepdims=True) / 7).astype(np.float16).astype(np.float64)
    return (np.clip(np.rint(x / np.where(s > 0, s, np.inf)), -7, 7) * s).reshape(x.shape[:-2] + (D,))


def _exact_rotated(x, at, rope_table):
    """numpy f64, rounded to f16 as the cache and the query hold it."""
    cis = rope_table.cpu().double().numpy()[at][..., None, :, :]
    x = x.cpu().double().numpy()
    z = (x[..., :64] + 1j * x[..., 64:]) * (cis[..., 0] + 1j * cis[..., 1])
    return torch.from_numpy(np.concatenate([z.real, z.imag], -1).astype(np.float16))


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "logprobs":
        x = st["logits"].double()
        lse = torch.logsumexp(x, -1)
        lp = torch.where((lse > -math.inf)[:, None], x - lse[:, None], torch.full_like(x, -math.inf))
        h = -torch.nan_to_num(lp.exp() * lp, nan=0.0).sum(-1)
        rows, order = st["logits"].float().cpu().numpy(), []
        for r in rows:  # value down, index up
            order.append(np.lexsort((np.arange(len(r)), -r))[:case["top"]])
        ids = torch.from_numpy(np.stack(order)).cuda()
        return {"logprob": lp[torch.arange(len(rows)), st["tokens"].long()], "entropy": h, "ids": ids.int(),
                "top": torch.take_along_dim(lp, ids, 1)}
    if op == "pages":
        if case["kv"] == "f16":
            return None  # bytes moved: nothing is computed
        src = st["from"]
        return {"k": _exact_rows(st["k_pool"][src], False).permute(0, 2, 3, 1, 4).flatten(1, 2),
                "v": _exact_rows(st["v_pool"][src], True).permute(0, 2, 3, 1, 4).flatten(1, 2)}
    starts = st["starts"].cpu().numpy()
    if op == "append":
        k = st["new_k"]
        if case["rope"]:
            k = _exact_rotated(k, starts[:, None] + np.arange(case["tokens"]), st["rope_table"])
        return {"k": _exact_held(k), "v": _exact_held(st["new_v"])}
    b, h, g = case["batch"], case["heads"], case["kv_heads"]
    q = _exact_rotated(st["q"], starts, st["rope_table"]).cuda() if case["rope"] else st["q"]
    nk = _exact_rotated(st["new_k"], starts, st["rope_table"]) if case["rope"] else st["new_k"]
    nk, nv = _exact_held(nk), _exact_held(st["new_v"])
    out = torch.zeros((b, h, D), dtype=torch.float64, device="cuda")
    for i, n in enumerate(st["lengths"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        pages = st["table"][i, :-(-n // case["page"])].long()
        k, v = (_exact_rows(st[p][pages], p == "v_pool").permute(0, 2, 3, 1, 4).reshape(-1, g, D)
                for p in ("k_pool", "v_pool"))
        if case["append"]:
            k[n - 1], v[n - 1] = torch.from_numpy(nk[i]).cuda(), torch.from_numpy(nv[i]).cuda()
        x = torch.einsum("gud,tgd->gut", q[i].double().view(g, h // g, D), k[first:n]) / math.sqrt(D)
        if case["softcap"]:
            x = case["softcap"] * torch.tanh(x / case["softcap"])
        out[i] = torch.einsum("gut,tgd->gud", torch.softmax(x, -1), v[first:n]).reshape(h, D)
    return {"out": out, "k": nk[:, None], "v": nv[:, None]} if case["append"] else {"out": out}
