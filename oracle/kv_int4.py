"""numpy restatement of the 4-bit KV cache, its attention and the token log
probabilities, from their definitions (int4 rows: per token, kv head and 32
dims s = f16(max|x| / 7), n = clamp(rint(x / s), -7, 7) + 8).  Quantisation in
IEEE f32 (bytes are compared exactly), attention and log probabilities in f64.
"""
from __future__ import annotations

import numpy as np

GROUPS, BLOCK = 4, 1152


def quantize(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """f16 rows [..., 128] -> f16 scales [..., 4], codes n uint8 [..., 128]."""
    x = np.asarray(x, np.float16).astype(np.float32)
    g = x.reshape(x.shape[:-1] + (GROUPS, 32))
    s = (np.abs(g).max(-1) / np.float32(7)).astype(np.float16)
    sf = s.astype(np.float32)[..., None]
    q = np.rint(np.divide(g, sf, out=np.zeros_like(g), where=sf != 0))
    return s, (np.clip(q, -7, 7) + 8).astype(np.uint8).reshape(x.shape)


def values(s: np.ndarray, n: np.ndarray) -> np.ndarray:
    """Scales and codes -> f64 values [..., 128]."""
    g = (n.astype(np.float64) - 8).reshape(n.shape[:-1] + (GROUPS, 32))
    return (g * s.astype(np.float64)[..., None]).reshape(n.shape)


def put(pool: np.ndarray, is_v: bool, page: int, head: int, in_page: int, s: np.ndarray, n: np.ndarray) -> None:
    """Writes one row's scales [4] and codes [128] into pool [pages, Hkv, page / 16, 1152]."""
    blk = pool[page, head, in_page // 16]
    tok = in_page % 16
    codes = blk[:1024].view(np.uint16)
    scales = blk[1024:].view(np.float16)
    for g in range(GROUPS):
        d = n[32 * g:32 * g + 32].astype(np.uint16)
        if is_v:
            for r in range(8):
                at = ((((tok >> 3) * 8 + r) * 4 + ((tok >> 1) & 3)) * GROUPS + g) * 2 + (tok & 1)
                codes[at] = d[4 * r] | d[4 * r + 1] << 4 | d[4 * r + 2] << 8 | d[4 * r + 3] << 12
            scales[((tok >> 1) * GROUPS + g) * 2 + (tok & 1)] = s[g]
        else:
            for t in range(4):
                at = ((tok * 4 + t) * GROUPS + g) * 2
                e = d[8 * t:8 * t + 8]
                codes[at] = e[0] | e[2] << 4 | e[4] << 8 | e[6] << 12
                codes[at + 1] = e[1] | e[3] << 4 | e[5] << 8 | e[7] << 12
            scales[tok * GROUPS + g] = s[g]


def get(pool: np.ndarray, is_v: bool, page: int, head: int, in_page: int) -> np.ndarray:
    """One row's f64 values."""
    blk = np.ascontiguousarray(pool[page, head, in_page // 16])
    tok = in_page % 16
    codes, scales = blk[:1024].view(np.uint16), blk[1024:].view(np.float16)
    out = np.empty(128)
    for g in range(GROUPS):
        if is_v:
            s = float(scales[((tok >> 1) * GROUPS + g) * 2 + (tok & 1)])
            for r in range(8):
                at = ((((tok >> 3) * 8 + r) * 4 + ((tok >> 1) & 3)) * GROUPS + g) * 2 + (tok & 1)
                for i in range(4):
                    out[32 * g + 4 * r + i] = (int(codes[at] >> (4 * i) & 15) - 8) * s
        else:
            s = float(scales[tok * GROUPS + g])
            for t in range(4):
                at = ((tok * 4 + t) * GROUPS + g) * 2
                for i in range(8):
                    out[32 * g + 8 * t + i] = (int(codes[at + (i & 1)] >> (4 * (i >> 1)) & 15) - 8) * s
    return out


def rotate(x: np.ndarray, pos: np.ndarray, freq_cis: np.ndarray) -> np.ndarray:
    """RoPE of f16 rows x [..., heads, 128] at pos [...]: products and sums rounded in f32, result f16."""
    cis = freq_cis[pos][..., None, :, :].astype(np.float32)
    c, s = cis[..., 0], cis[..., 1]
    f = x.astype(np.float32)
    x0, x1 = f[..., :64], f[..., 64:]
    return np.concatenate([x0 * c - x1 * s, x0 * s + x1 * c], -1).astype(np.float16)


def append(k_pool, v_pool, table, page_size, new_k, new_v, positions, freq_cis=None) -> None:
    """new_k / new_v [B, T, Hkv, 128] f16 at positions[b] + t (mapped rows only)."""
    B, T, H, _ = new_k.shape
    if freq_cis is not None:
        new_k = rotate(new_k, positions[:, None] + np.arange(T), freq_cis)
    for pool, rows, is_v in ((k_pool, new_k, False), (v_pool, new_v, True)):
        s, n = quantize(rows)
        for b in range(B):
            for t in range(T):
                p = int(positions[b]) + t
                if p < 0 or p // page_size >= table.shape[1]:
                    continue
                page = int(table[b, p // page_size])
                if not 0 <= page < pool.shape[0]:
                    continue
                for h in range(H):
                    put(pool, is_v, page, h, p % page_size, s[b, t, h], n[b, t, h])


def rows(pool, is_v, table_row, page_size, count) -> np.ndarray:
    """The first `count` tokens of a sequence: f64 [count, Hkv, 128]."""
    return np.stack([np.stack([get(pool, is_v, int(table_row[p // page_size]), h, p % page_size)
                               for h in range(pool.shape[1])]) for p in range(count)])


def attend(q, k, v, scale, window=0, softcap=0.0):
    """q [H, 128], k / v [L, Hkv, 128] f64 -> (out [H, 128], the same with |v|): one query after L tokens."""
    H, L, G = q.shape[0], k.shape[0], k.shape[1]
    if L == 0:
        return np.zeros((H, 128)), np.zeros((H, 128))
    lo = max(0, L - window) if window else 0
    k, v = k[lo:], v[lo:]
    x = np.einsum("gud,tgd->gut", q.astype(np.float64).reshape(G, H // G, 128), k) * scale
    if softcap:
        x = softcap * np.tanh(x / softcap)
    e = np.exp(x - x.max(-1, keepdims=True))
    p = e / e.sum(-1, keepdims=True)
    return tuple(np.einsum("gut,tgd->gud", p, w).reshape(H, 128) for w in (v, np.abs(v)))


def logprobs(x: np.ndarray, tokens: np.ndarray, top_k: int):
    """x [rows, vocab] -> logprob, entropy (f64), top ids, top logprobs."""
    x = x.astype(np.float64)
    n = len(x)
    lp = np.empty_like(x)
    h = np.empty(n)
    for r in range(n):
        m = x[r].max()
        if m == -np.inf:
            lp[r], h[r] = -np.inf, 0.0
            continue
        if not np.isfinite(m):  # +inf or NaN
            lp[r], h[r] = np.nan, np.nan
            continue
        lp[r] = x[r] - m - np.log(np.exp(x[r] - m).sum())
        p = np.exp(lp[r])
        h[r] = -(p[p > 0] * lp[r][p > 0]).sum()
    order = np.where(np.isnan(x), -np.inf, x)
    ids = np.stack([np.lexsort((np.arange(x.shape[1]), -r))[:top_k] for r in order]) if n else np.zeros((0, top_k))
    return lp[np.arange(n), tokens], h, ids, np.take_along_axis(lp, ids, 1)
