"""GPU parity of the 4-bit paged KV cache: append and read (exact), attention.

Attention tolerance, from the kernel's roundings: every p and every product of
p with a V scale is rounded to f16 (2^-11 relative each at most), sums and
statistics are f32, scores are off by at most about 1e-5 (f32 accumulation of
128 products) and exponentials by 2^-22:
  |o - ref| <= 2^-10 (1 + 2^-4) A + 2e-5 max|v|,  A = sum p |v| / sum p,
bf16 outputs are rounded once more (2^-8 |ref|).
"""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from doe_b200 import ops
from doe_b200._abi import DOE_DEVICE_ERR_LENGTH, DOE_DEVICE_ERR_PAGE, DOE_DEVICE_ERR_POSITION, DoeError
from doe_b200.decoder import rope_table
from doe_b200.kv import PagedKVCache
from oracle import kv_int4

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def _t(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _table(g, lens, page, spare=1):
    need = [-(-int(n) // page) for n in lens]
    total = sum(need) + spare
    perm = g.permutation(total).astype(np.int32)
    table = np.full((len(lens), max(need) + 1), -1, np.int32)
    o = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[o:o + n]
        o += n
    return table, total


def _rows(g, shape, std=1.0):
    return (g.standard_normal(shape) * std).astype(np.float16)


class Case:
    """Sequences of `lens` tokens in an int4 cache, filled through the oracle."""

    def __init__(self, seed, lens, Hkv=2, group=4, page=16, std=1.0, vstd=1.0):
        g = self.g = np.random.default_rng(seed)
        self.lens, self.Hkv, self.H, self.page = np.asarray(lens, np.int32), Hkv, Hkv * group, page
        self.table, self.pages = _table(g, self.lens, page)
        B, T = len(lens), int(max(lens))
        self.k, self.v = _rows(g, (B, T, Hkv, 128), std), _rows(g, (B, T, Hkv, 128), vstd)
        # unwritten bytes hold anything, also scales that are infinite or NaN
        self.kp, self.vp = (g.integers(0, 256, (self.pages, Hkv, page // 16, 1152)).astype(np.uint8) for _ in range(2))
        for b in range(B):
            n = int(self.lens[b])
            if n:
                kv_int4.append(self.kp, self.vp, self.table[b:b + 1], page, self.k[b:b + 1, :n], self.v[b:b + 1, :n],
                               np.zeros(1, np.int64))
        self.q = _rows(g, (B, self.H, 128))

    def cache(self):
        return PagedKVCache.from_pools(_t(self.kp), _t(self.vp), page_size=self.page, num_kv_heads=self.Hkv,
                                       head_dim=128, block_table=_t(self.table), kv_dtype="int4")

    def values(self, b, k=None, v=None):
        out = []
        for x in (self.k if k is None else k, self.v if v is None else v):
            out.append(kv_int4.values(*kv_int4.quantize(x[b, :self.lens[b]])))
        return out

    def check(self, out, scale, window=0, softcap=0.0, q=None, k=None, v=None, bf16=False):
        q = self.q if q is None else q
        for b in range(len(self.lens)):
            kk, vv = self.values(b, k, v)
            ref, a = kv_int4.attend(q[b], kk, vv, scale, window, softcap)
            bound = 2.0 ** -10 * (1 + 2.0 ** -4) * a + 2e-5 * (np.abs(vv).max() if len(vv) else 0.0) + 1e-30
            if bf16:
                bound = bound + 2.0 ** -8 * np.abs(ref)
            err = np.abs(out[b].astype(np.float64) - ref)
            assert (err <= bound).all(), (b, self.lens[b], float((err / bound).max()))


def _decode(c, cache=None, **kw):
    status = ops.status_word()
    out = ops.paged_decode(cache or c.cache(), _t(c.q), _t(c.lens), kw.pop("scale", 128 ** -0.5), status=status, **kw)
    assert int(status.item()) == 0
    return out.float().cpu().numpy()


@pytest.mark.parametrize("Hkv,group", [(1, 1), (2, 2), (1, 3), (2, 4), (1, 5), (1, 6), (1, 7), (2, 8)])
def test_decode_head_groups(Hkv, group):
    c = Case(Hkv * 10 + group, [0, 1, 2, 15, 16, 17, 33, 64, 65, 300], Hkv, group)
    c.check(_decode(c), 128 ** -0.5)


@pytest.mark.parametrize("page", [16, 32, 48, 64])
@pytest.mark.parametrize("split_pages", [0, 1, 3])
def test_decode_pages_and_splits(page, split_pages):
    c = Case(page + split_pages, [1, 47, 48, 49, 700, 0, 129], 2, 4, page)
    out = _decode(c, split_pages=split_pages)
    c.check(out, 128 ** -0.5)
    assert np.array_equal(out, _decode(c, split_pages=split_pages)), "results depend on timing"


@pytest.mark.parametrize("window,softcap", [(1, 0.0), (16, 0.0), (17, 30.0), (100, 0.0), (5000, 5.0), (0, 50.0)])
def test_decode_window_and_softcap(window, softcap):
    c = Case(window, [0, 1, 16, 17, 99, 100, 101, 257], 1, 4)
    c.check(_decode(c, sliding_window=window, softcap=softcap, scale=0.3), 0.3, window, softcap)
    c.check(_decode(c, sliding_window=window, softcap=softcap, scale=0.3, split_pages=2), 0.3, window, softcap)


@pytest.mark.parametrize("std,vstd,scale", [(1.0, 1e-4, 0.1), (1.0, 3e-6, 0.1), (1.0, 900.0, 0.1), (6.0, 12000.0, 0.2),
                                            (100.0, 1.0, 1.0), (1e-3, 1.0, 0.1), (1.0, 1.0, 0.0)])
def test_decode_magnitudes(std, vstd, scale):
    """V from f16's subnormals to its largest values, one-hot and flat softmaxes."""
    c = Case(7, [1, 40, 333], 1, 4, std=std, vstd=vstd)
    c.v = np.clip(c.v.astype(np.float32), -65504, 65504).astype(np.float16)
    c = _refill(c)
    out = _decode(c, scale=scale)
    assert np.isfinite(out).all()
    # scores of hundreds are off by 2^-23 of their size
    for b in range(3):
        kk, vv = c.values(b)
        ref, a = kv_int4.attend(c.q[b], kk, vv, scale)
        sc = np.abs(np.einsum("hd,td->ht", np.abs(c.q[b].astype(np.float64)), np.abs(kk[:, 0]))).max() * scale
        bound = (2.0 ** -10 * (1 + 2.0 ** -4) + sc * 2.0 ** -22) * a + 2e-5 * np.abs(vv).max()
        assert (np.abs(out[b] - ref) <= bound).all()


def _refill(c):
    for b in range(len(c.lens)):
        n = int(c.lens[b])
        kv_int4.append(c.kp, c.vp, c.table[b:b + 1], c.page, c.k[b:b + 1, :n], c.v[b:b + 1, :n], np.zeros(1, np.int64))
    return c


def test_decode_reference_follows_scores_and_scales():
    """Scores that rise along the sequence and V scales that jump late."""
    c = Case(8, [400], 1, 4, std=0.2)
    ramp = np.linspace(0, 6, 400)[None, :, None, None]
    c.k = (np.sign(c.q[:, :1, None, :].transpose(0, 1, 2, 3)) * ramp).astype(np.float16).reshape(1, 400, 1, 128)
    c.v = c.v * np.where(np.arange(400) == 390, 2000.0, 0.05)[None, :, None, None].astype(np.float16)
    c.v = c.v.astype(np.float16)
    c = _refill(c)
    c.check(_decode(c, scale=0.3), 0.3)
    c.check(_decode(c, scale=-0.3, split_pages=1), -0.3)


@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("stable", [False, True])
def test_decode_fused_append(rope, stable):
    c = Case(21, [1, 2, 15, 16, 17, 31, 32, 33, 65, 300], 2, 4)
    B = len(c.lens)
    nk, nv = _rows(c.g, (B, 2, 128)), _rows(c.g, (B, 2, 128), 3.0)
    cis = rope_table(301, 128, 10000.0)
    last = c.lens.astype(np.int64) - 1
    rk, q = (kv_int4.rotate(nk, last, cis), kv_int4.rotate(c.q, last, cis)) if rope else (nk, c.q)
    cache = c.cache()
    out = _decode(c, cache, new_k=_t(nk), new_v=_t(nv), freq_cis=_t(cis) if rope else None, inputs_stable=stable,
                  split_pages=1)
    k, v = c.k.copy(), c.v.copy()
    for b in range(B):
        k[b, last[b]], v[b, last[b]] = rk[b], nv[b]
    c.check(out, 128 ** -0.5, q=q, k=k, v=v)
    kv_int4.append(c.kp, c.vp, c.table, 16, rk[:, None], nv[:, None], last)
    assert np.array_equal(cache.k_pool.cpu().numpy(), c.kp), "the append wrote other K bytes"
    assert np.array_equal(cache.v_pool.cpu().numpy(), c.vp), "the append wrote other V bytes"


def test_decode_bf16_and_kept_workspace():
    c = Case(22, [5, 700, 64], 2, 4)
    cache = c.cache()
    ws = ops.decode_workspace(cache, 3, c.H, split_pages=2)
    for _ in range(3):
        out = _decode(c, cache, split_pages=2, ws=ws, out_dtype=torch.bfloat16)
        c.check(out, 128 ** -0.5, bf16=True)


def test_decode_on_a_side_stream():
    c = Case(23, [260, 31], 1, 4)
    cache, q, n = c.cache(), _t(c.q), _t(c.lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = ops.paged_decode(cache, q, n, 128 ** -0.5, stream=s)
    s.synchronize()
    c.check(out.cpu().numpy(), 128 ** -0.5)


def test_decode_reports_bad_pages_and_lengths():
    c = Case(24, [40, 40], 1, 4)
    cache = c.cache()
    status = ops.status_word()
    table = c.table.copy()
    table[0, 1] = c.pages + 3
    cache.set_block_table(table)
    ops.paged_decode(cache, _t(c.q), _t(c.lens), 0.1, status=status)
    assert int(status.item()) == DOE_DEVICE_ERR_PAGE
    status.zero_()
    cache.set_block_table(c.table)
    long = c.lens.copy()
    long[1] = 10 ** 6  # clamped to the block table's row, which ends unmapped
    out = ops.paged_decode(cache, _t(c.q), _t(long), 128 ** -0.5, status=status)
    assert int(status.item()) & DOE_DEVICE_ERR_LENGTH
    ref, a = kv_int4.attend(c.q[0], *c.values(0), 128 ** -0.5)
    assert (np.abs(out[0].cpu().numpy() - ref) <= 2.0 ** -9 * a + 1e-4).all()
    status.zero_()
    neg = c.lens.copy()
    neg[0] = -5
    out = ops.paged_decode(cache, _t(c.q), _t(neg), 0.1, status=status)
    assert int(status.item()) == DOE_DEVICE_ERR_LENGTH and not out[0].any()


def test_decode_long_sequence_splits_and_far_pages():
    """130k tokens in 64-token pages: many splits per row, page walks across every prefetch register."""
    g = np.random.default_rng(3)
    n, page = 130001, 64
    np_pages = -(-n // page)
    cache = PagedKVCache(num_pages=np_pages, page_size=page, num_kv_heads=1, head_dim=128,
                         block_table=g.permutation(np_pages).astype(np.int32)[None], kv_dtype="int4")
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    k = torch.randn((1, n, 1, 128), generator=gen, device="cuda").half()
    v = torch.randn((1, n, 1, 128), generator=gen, device="cuda").half()
    ops.paged_append(cache, k, v, torch.zeros(1, dtype=torch.int32, device="cuda"))
    q = torch.randn((1, 8, 128), generator=gen, device="cuda").half()
    kk, vv = ops.paged_read(cache, torch.zeros(1, dtype=torch.int32, device="cuda"), n, dtype=torch.float32)
    x = (q[0].double() @ kk[0, :, 0].double().T) / 128 ** 0.5
    p = torch.softmax(x, -1)
    ref, a = p @ vv[0, :, 0].double(), p @ vv[0, :, 0].double().abs()
    for split in (0, 8, 100):
        out = ops.paged_decode(cache, q, torch.tensor([n], dtype=torch.int32, device="cuda"), 128 ** -0.5,
                               split_pages=split)[0].double()
        assert bool(((out - ref).abs() <= 2.0 ** -10 * 1.1 * a + 1e-4).all())


@pytest.mark.parametrize("batch", [1, 32])
def test_decode_long_flat_softmax_keeps_its_precision(batch):
    """Tens of thousands of about equal weights: O is a hundred times smaller than the sums of codes
    it comes from.  The two f16 roundings leave a relative error (2-norm) of 2^-12 each at most; 5e-4
    leaves as much again for the f32 sums."""
    n = 20000
    pages = -(-n // 16)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(batch, 1)  # one text, shared
    cache = PagedKVCache(num_pages=pages, page_size=16, num_kv_heads=8, head_dim=128, block_table=np.zeros((1, 1)),
                         kv_dtype="int4")
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    k, v = (torch.randn((1, n, 8, 128), generator=g, device="cuda").half() for _ in range(2))
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache.block_table, cache.max_pages_per_seq = table, pages
    ops.paged_append(cache, k, v, zero)
    q = torch.randn((batch, 32, 128), generator=g, device="cuda").half()
    out = ops.paged_decode(cache, q, torch.full((batch,), n, dtype=torch.int32, device="cuda"), 128 ** -0.5).double()
    k, v = (x[0].double() for x in ops.paged_read(cache, zero, n, dtype=torch.float32))
    x = torch.einsum("bgud,tgd->bgut", q.double().view(batch, 8, 4, 128), k) / 128 ** 0.5
    ref = torch.einsum("bgut,tgd->bgud", torch.softmax(x, -1), v).reshape(batch, 32, 128)
    assert float((out - ref).norm() / ref.norm()) < 5e-4


@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("Hkv,page,T", [(1, 16, 1), (2, 16, 2), (8, 16, 15), (2, 32, 16), (1, 48, 17), (4, 16, 50), (3, 64, 33)])
def test_append_is_exact(Hkv, page, T, rope):
    g = np.random.default_rng(T)
    starts = np.array([0, 1, 7, 8, 15, 16, 31, 90], np.int32)
    table, pages = _table(g, starts + T, page)
    k, v = _rows(g, (8, T, Hkv, 128), 2.0), _rows(g, (8, T, Hkv, 128), 0.01)
    k[0, 0] = 0
    v[1, 0, 0, :40] = 65504
    v[2, 0, 0] = 6e-8
    k[3, 0, 0, :7] = np.array([7, 0.5, 1.5, 2.5, -0.5, -1.5, 6.5])  # ties where that group's scale is 1
    k[3, 0, 0, 7:32] = 0
    cis = rope_table(200, 128, 10000.0) if rope else None
    kp, vp = (g.integers(0, 256, (pages, Hkv, page // 16, 1152)).astype(np.uint8) for _ in range(2))
    cache = PagedKVCache.from_pools(_t(kp), _t(vp), page_size=page, num_kv_heads=Hkv, head_dim=128,
                                    block_table=_t(table), kv_dtype="int4")
    status = ops.status_word()
    ops.paged_append(cache, _t(k), _t(v), _t(starts), status=status, freq_cis=_t(cis) if rope else None)
    kv_int4.append(kp, vp, table, page, k, v, starts.astype(np.int64), cis)
    assert int(status.item()) == 0
    assert np.array_equal(cache.k_pool.cpu().numpy(), kp)
    assert np.array_equal(cache.v_pool.cpu().numpy(), vp)
    # and back, as values: exact in f32, rounded once in f16 and bf16
    rk = kv_int4.rotate(k, starts[:, None] + np.arange(T), cis) if rope else k
    want = [kv_int4.values(*kv_int4.quantize(x)) for x in (rk, v)]
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        got = ops.paged_read(cache, _t(starts), T, dtype=dt, status=status)
        for a, w in zip(got, want):
            assert torch.equal(a.cpu(), torch.from_numpy(w.astype(np.float32)).to(dt))
    assert int(status.item()) == 0


def test_append_every_scale_and_code():
    """Rows over f16's whole exponent range, so scales reach its subnormals, zero and 9358."""
    g = np.random.default_rng(5)
    mag = 2.0 ** np.linspace(-25, 16, 512)
    k = np.clip(g.standard_normal((1, 512, 1, 128)) * mag[None, :, None, None], -65504, 65504).astype(np.float16)
    v = (g.integers(-14, 15, (1, 512, 1, 128)) / 2 * mag[::-1][None, :, None, None] / 16).astype(np.float16)  # ties
    table, pages = _table(g, [512], 16)
    cache = PagedKVCache(num_pages=pages, page_size=16, num_kv_heads=1, head_dim=128, block_table=table, kv_dtype="int4")
    kp, vp = (np.zeros((pages, 1, 1, 1152), np.uint8) for _ in range(2))
    ops.paged_append(cache, _t(k), _t(v), torch.zeros(1, dtype=torch.int32, device="cuda"))
    kv_int4.append(kp, vp, table, 16, k, v, np.zeros(1, np.int64))
    assert np.array_equal(cache.k_pool.cpu().numpy(), kp)
    assert np.array_equal(cache.v_pool.cpu().numpy(), vp)


def test_append_skips_and_read_zeroes_unmapped_rows():
    g = np.random.default_rng(6)
    table = np.array([[0, -1], [1, 2], [3, 3]], np.int32)
    cache = PagedKVCache(num_pages=3, page_size=16, num_kv_heads=2, head_dim=128, block_table=table, kv_dtype="int4")
    k, v = _rows(g, (3, 20, 2, 128)), _rows(g, (3, 20, 2, 128))
    starts = np.array([4, 30, -1], np.int32)  # runs into unmapped pages, off the table, negative
    kp, vp = (np.zeros((3, 2, 1, 1152), np.uint8) for _ in range(2))
    status = ops.status_word()
    ops.paged_append(cache, _t(k), _t(v), _t(starts), status=status)
    assert int(status.item()) == DOE_DEVICE_ERR_PAGE
    kv_int4.append(kp, vp, table[:2], 16, k[:2], v[:2], starts[:2].astype(np.int64))
    assert np.array_equal(cache.k_pool.cpu().numpy(), kp) and np.array_equal(cache.v_pool.cpu().numpy(), vp)
    status.zero_()
    out = [torch.full((3, 20, 2, 128), 9.0, device="cuda") for _ in range(2)]
    ops.paged_read(cache, _t(starts), 20, dtype=torch.float32, out=out, status=status)
    assert int(status.item()) == DOE_DEVICE_ERR_PAGE
    got = out[0].cpu().numpy()
    want = kv_int4.values(*kv_int4.quantize(k))
    assert np.array_equal(got[0, :12], want[0, :12].astype(np.float32)) and (got[0, 12:] == 0).all()
    assert np.array_equal(got[1, :2], want[1, :2].astype(np.float32)) and (got[1, 2:] == 0).all()
    assert (got[2] == 0).all()
    old = PagedKVCache(num_pages=1, page_size=16, num_kv_heads=1, head_dim=128, block_table=np.array([[0, -1]]))
    old.k_pool.fill_(2.0)
    got = ops.paged_read(old, _t(np.array([10], np.int32)), 12, status=status)[0]
    assert (got[0, :6] == 2).all() and (got[0, 6:] == 0).all()


def test_append_rope_beyond_the_table_reports():
    cache = PagedKVCache(num_pages=2, page_size=16, num_kv_heads=1, head_dim=128, block_table=np.array([[0, 1]]),
                         kv_dtype="int4")
    k = torch.ones((1, 4, 1, 128), dtype=torch.float16, device="cuda")
    status = ops.status_word()
    ops.paged_append(cache, k, k, torch.tensor([8], dtype=torch.int32, device="cuda"), status=status,
                     freq_cis=_t(rope_table(10, 128, 10000.0)))
    assert int(status.item()) == DOE_DEVICE_ERR_POSITION


@pytest.mark.parametrize("kv_dtype", ["f16", "int8"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_read_of_f16_and_int8_caches(kv_dtype, D):
    g = np.random.default_rng(D)
    starts, T = np.array([0, 3, 16, 40], np.int32), 19
    table, pages = _table(g, starts + T, 16)
    cache = PagedKVCache(num_pages=pages, page_size=16, num_kv_heads=3, head_dim=D, block_table=table, kv_dtype=kv_dtype)
    k, v = _rows(g, (4, T, 3, D)), _rows(g, (4, T, 3, D), 5.0)
    ops.paged_append(cache, _t(k), _t(v), _t(starts))
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        got = ops.paged_read(cache, _t(starts), T, dtype=dt)
        for a, x in zip(got, (k, v)):
            w = torch.from_numpy(x).float()
            if kv_dtype == "int8":
                s = (w.abs().amax(-1, keepdim=True) / 127).half().float()
                w = torch.clamp(torch.round(w / s), -127, 127) * s
            assert torch.equal(a.cpu(), w.to(dt))


def test_refusals():
    cache = PagedKVCache(num_pages=2, page_size=16, num_kv_heads=1, head_dim=128, block_table=np.array([[0, 1]]),
                         kv_dtype="int4")
    with pytest.raises(DoeError):
        ops.paged_gather(cache, 0, 0, 4)
    with pytest.raises(ValueError):
        ops.paged_read(cache, torch.zeros(2, dtype=torch.int32, device="cuda"), 1)  # two sequences, one table row
    with pytest.raises(ValueError):
        ops.paged_read(cache, torch.zeros(1, dtype=torch.int32, device="cuda"), 1, dtype=torch.int8)
    with pytest.raises(ValueError):
        PagedKVCache(num_pages=2, page_size=16, num_kv_heads=1, head_dim=64, block_table=np.array([[0]]), kv_dtype="int4")
    with pytest.raises(ValueError):
        PagedKVCache.from_pools(cache.k_pool[:1], cache.v_pool, page_size=16, num_kv_heads=1, head_dim=128,
                                block_table=cache.block_table, kv_dtype="int4")
    with pytest.raises(ValueError):
        PagedKVCache.from_pools(cache.k_pool, cache.v_pool, page_size=16, num_kv_heads=1, head_dim=128,
                                block_table=cache.block_table.cpu(), kv_dtype="int4")


def test_non_finite_rows_stay_non_finite():
    """A NaN anywhere in a group makes the group's scale NaN, so it reads back as NaN; an infinity
    reads back as infinities and NaNs.  The other groups, heads and tokens keep their values, and a
    decode sees the NaNs exactly where the row is attended."""
    g = np.random.default_rng(9)
    n, Hkv = 70, 2
    table, pages = _table(g, [n], 16)
    k, v = _rows(g, (1, n, Hkv, 128)), _rows(g, (1, n, Hkv, 128))
    clean = [kv_int4.values(*kv_int4.quantize(x)).astype(np.float32) for x in (k, v)]
    k[0, 3, 0, 40] = np.nan
    v[0, 5, 1, 127] = np.nan
    v[0, 2, 1, 0] = -np.inf
    k[0, 6, 1, 64] = np.inf
    cache = PagedKVCache(num_pages=pages, page_size=16, num_kv_heads=Hkv, head_dim=128, block_table=table,
                         kv_dtype="int4")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.paged_append(cache, _t(k), _t(v), zero)
    for dt in (torch.float32, torch.float16):
        rk, rv = (x.float().cpu().numpy() for x in ops.paged_read(cache, zero, n, dtype=dt))
        assert np.isnan(rk[0, 3, 0, 32:64]).all() and np.isnan(rv[0, 5, 1, 96:]).all()
        assert not np.isfinite(rv[0, 2, 1, :32]).any() and not np.isfinite(rk[0, 6, 1, 64:96]).any()
        for r, w in zip((rk, rv), clean):
            bad = ~np.isfinite(r)
            w = torch.from_numpy(w).to(dt).float().numpy()
            assert bad.sum() == 64 and np.array_equal(r[~bad], w[~bad])
    q = _t(_rows(g, (1, 8, 128)))
    length = torch.full((1,), n, dtype=torch.int32, device="cuda")
    out = ops.paged_decode(cache, q, length, 0.1)[0].cpu().numpy()
    assert np.isnan(out[:4]).all() and not np.isfinite(out[4:, 96:]).any()
    # past the window
    out = ops.paged_decode(cache, q, length, 0.1, sliding_window=n - 7)[0].cpu().numpy()
    ref, a = kv_int4.attend(q[0].cpu().numpy(), clean[0][0], clean[1][0], 0.1, n - 7)
    assert (np.abs(out - ref) <= 2.0 ** -10 * (1 + 2.0 ** -4) * a + 2e-5 * np.abs(clean[1]).max()).all()


def test_decode_appends_non_finite_rows_as_such():
    c = Case(31, [20, 33], 2, 4)
    cache = c.cache()
    nk, nv = _rows(c.g, (2, 2, 128)), _rows(c.g, (2, 2, 128))
    nk[0, 1, 33] = np.nan
    nv[1, 0, 70] = np.nan
    out = _decode(c, cache, new_k=_t(nk), new_v=_t(nv))
    assert np.isnan(out[0, 4:]).all() and np.isfinite(out[0, :4]).all()
    assert np.isnan(out[1, :4, 64:96]).all() and np.isfinite(out[1, 4:]).all()
    k, v = (x.cpu().numpy() for x in ops.paged_read(cache, _t(c.lens - 1), 1, dtype=torch.float32))
    assert np.isnan(k[0, 0, 1, 32:64]).all() and np.isnan(k).sum() == 32
    assert np.isnan(v[1, 0, 0, 64:96]).all() and np.isnan(v).sum() == 32


@pytest.mark.parametrize("width", [1, 300])
@pytest.mark.parametrize("lens", [[4000], [300, 0, 4097, 1], [17] * 20 + [2500], [0] * 40 + [900, 33, 2000]])
@pytest.mark.parametrize("Hkv", [1, 3])
def test_decode_few_rows_share_the_splits_by_length(lens, width, Hkv):
    """Splits follow the lengths, not the block table's width (`width` unused pages a row)."""
    c = Case(len(lens) + width, lens, Hkv, 4)
    c.table = np.concatenate([c.table, np.full((len(lens), width), -1, np.int32)], 1)
    out = _decode(c)
    c.check(out, 128 ** -0.5)
    assert np.array_equal(out, _decode(c)), "results depend on timing"
    c.check(_decode(c, sliding_window=1000), 128 ** -0.5, 1000)


def test_refusals_of_shapes():
    cache = PagedKVCache(num_pages=2, page_size=16, num_kv_heads=2, head_dim=128, block_table=np.array([[0, 1]]),
                         kv_dtype="int4")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    f16 = lambda *s: torch.zeros(s, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError):
        ops.paged_decode(cache, f16(2, 4, 128), i32(1, 1), 0.1)  # two sequences, one table row
    with pytest.raises(ValueError):
        ops.paged_decode(cache, f16(1, 4, 128), i32(1, 1), 0.1)
    with pytest.raises(ValueError):
        ops.paged_decode(cache, f16(1, 4, 64), i32(1), 0.1)
    with pytest.raises(ValueError):
        ops.paged_decode(cache, f16(1, 4, 128), i32(1), 0.1, new_k=f16(1, 1, 128), new_v=f16(1, 2, 128))
    with pytest.raises(DoeError):
        ops.paged_decode(cache, f16(1, 3, 128), i32(1), 0.1)  # 3 heads, 2 kv heads
    with pytest.raises(DoeError):
        ops.paged_decode(cache, f16(1, 18, 128), i32(1), 0.1)  # 9 heads per kv head
    with pytest.raises(ValueError):
        ops.paged_append(cache, f16(1, 3, 2, 128), f16(1, 3, 1, 128), i32(0))
    with pytest.raises(ValueError):
        ops.paged_append(cache, f16(1, 3, 2, 128), f16(1, 3, 2, 128), i32(0, 0))
    with pytest.raises(ValueError):
        ops.paged_append(cache, f16(2, 3, 2, 128), f16(2, 3, 2, 128), i32(0, 0))


def test_backend_dispatch_of_an_int4_cache():
    """kv_append_paged and attention_paged_decode with kv_dtype 2 give the operators' bytes."""
    from doe_b200._abi import DOE_KV_INT4
    from doe_b200.backend import Bind, CudaBackend

    c = Case(41, [10, 200, 33], 2, 4)
    B, T, Hkv, H = 3, 5, c.Hkv, c.H
    nk, nv = _rows(c.g, (B, T, Hkv, 128)), _rows(c.g, (B, T, Hkv, 128))
    starts = c.lens - T
    cache = c.cache()
    ops.paged_append(cache, _t(nk), _t(nv), _t(starts))
    want = ops.paged_decode(cache, _t(c.q), _t(c.lens), 0.1).cpu().numpy()
    be = CudaBackend(0)
    try:
        scale = int(np.float32(0.1).view(np.uint32))
        uni = lambda *v: np.array(v, np.uint32)
        for h, a in ((1, uni(B, T, Hkv, 128, 16, c.pages, c.table.shape[1], DOE_KV_INT4)), (2, nk), (3, nv), (4, c.kp),
                     (5, c.vp), (6, c.table), (7, starts), (8, c.lens), (9, c.q),
                     (10, uni(B, H, Hkv, 128, 16, c.pages, c.table.shape[1], DOE_KV_INT4, scale, 0))):
            be.execute_buffer_write_bytes(h, 0, np.ascontiguousarray(a))
        be.execute_kernel_dispatch("kv_append_paged", [Bind(0, 1, size=32)] + [Bind(i, i + 1) for i in range(1, 7)])
        be.execute_kernel_dispatch("attention_paged_decode", [
            Bind(0, 10, size=40), Bind(1, 9), Bind(2, 4), Bind(3, 5), Bind(4, 6), Bind(5, 8),
            Bind(6, 11, size=B * H * 128 * 4)])
        out = np.frombuffer(be.capture_buffer(11, 0, B * H * 128 * 4), np.float32).reshape(want.shape)
        kp = np.frombuffer(be.capture_buffer(4, 0, c.kp.nbytes), np.uint8).reshape(c.kp.shape)
    finally:
        be.close()
    assert np.array_equal(kp, cache.k_pool.cpu().numpy())
    assert np.array_equal(out, want)


def test_a_captured_step_replays():
    """Append, decode, read back, a page copy and the log probabilities in one CUDA graph."""
    c = Case(51, [40, 3], 2, 4)
    cache = c.cache()
    g = np.random.default_rng(52)
    nk, nv, q = _t(_rows(g, (2, 2, 128))), _t(_rows(g, (2, 2, 128))), _t(c.q)
    chunk = _t(_rows(g, (2, 3, 2, 128)))
    lens, zero = _t(c.lens), _t(np.zeros(2, np.int32))
    logits, tokens = torch.randn((2, 5000), device="cuda"), torch.tensor([4, 9], dtype=torch.int32, device="cuda")
    spare = next(p for p in range(c.pages) if p not in c.table)
    pair = np.array([[int(c.table[0, 0]), spare]], np.int32)

    def step(cache):
        ops.paged_append(cache, chunk, chunk, zero)
        out = ops.paged_decode(cache, q, lens, 0.1, new_k=nk, new_v=nv)
        ops.paged_copy_pages(cache, pair)
        return (out, *ops.paged_read(cache, zero, 3), *ops.token_logprobs(logits, tokens, top_k=3), cache.k_pool.clone())

    want = [x.clone() for x in step(c.cache())]
    step(cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_decodes_of_any_shapes_share_a_stream():
    """2400 rows in clusters of 8, whose counters outgrow the region that all shapes have in common,
    between small decodes."""
    big = Case(61, [1] * 260 + [200] * 40, 8, 1)
    big.table = np.concatenate([big.table, np.full((300, 30), -1, np.int32)], 1)
    small = Case(62, [5000, 300], 2, 4)
    cb, cs = big.cache(), small.cache()
    first, alone = _decode(big, cb, split_pages=1), _decode(small, cs)
    big.check(first, 128 ** -0.5)
    small.check(alone, 128 ** -0.5)
    for _ in range(2):
        assert np.array_equal(_decode(small, cs), alone)
        assert np.array_equal(_decode(big, cb, split_pages=1), first)


def test_a_captured_decode_does_not_use_the_streams_workspace():
    """A graph captured on a stream that has decoded before, replayed beside decodes on that stream."""
    c = Case(71, [3000, 2500], 2, 4)
    cache, q, n = c.cache(), _t(c.q), _t(c.lens)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        want = ops.paged_decode(cache, q, n, 0.1).clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = ops.paged_decode(cache, q, n, 0.1)
    outs = []
    for _ in range(20):
        with torch.cuda.stream(other):
            graph.replay()
        with torch.cuda.stream(side):
            outs.append(ops.paged_decode(cache, q, n, 0.1))
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all(torch.equal(o, want) for o in outs)


def test_pools_and_pages_past_32_bit_offsets():
    """4.3 GB pools: pages around the 2^31st and 2^32nd byte and the last ones."""
    g = np.random.default_rng(81)
    pages, n = 3_740_000, 100
    cache = PagedKVCache(num_pages=pages, page_size=16, num_kv_heads=1, head_dim=128, block_table=np.zeros((1, 7)),
                         kv_dtype="int4")
    assert cache.k_pool.numel() > 2 ** 32
    edge = [2 ** 31 // 1152, 2 ** 32 // 1152]
    ids = [edge[0], edge[0] + 1, edge[1], edge[1] + 1, pages - 1, 0, pages - 2]
    cache.set_block_table(np.array([ids], np.int32))
    k, v, q = _rows(g, (1, n, 1, 128)), _rows(g, (1, n, 1, 128)), _rows(g, (1, 4, 128))
    zero, length = _t(np.zeros(1, np.int32)), _t(np.array([n], np.int32))
    status = ops.status_word()
    ops.paged_append(cache, _t(k), _t(v), zero, status=status)
    want = [kv_int4.values(*kv_int4.quantize(x)) for x in (k, v)]
    for a, w in zip(ops.paged_read(cache, zero, n, dtype=torch.float32, status=status), want):
        assert np.array_equal(a.cpu().numpy(), w.astype(np.float32))
    out = ops.paged_decode(cache, _t(q), length, 0.1, status=status)[0].cpu().numpy()
    ref, a = kv_int4.attend(q[0], want[0][0], want[1][0], 0.1)
    assert (np.abs(out - ref) <= 2.0 ** -10 * (1 + 2.0 ** -4) * a + 2e-5 * np.abs(want[1]).max()).all()
    ops.paged_copy_pages(cache, np.array([[i, 100 + j] for j, i in enumerate(ids)], np.int32))
    cache.set_block_table(np.arange(100, 107, dtype=np.int32)[None])
    assert np.array_equal(ops.paged_decode(cache, _t(q), length, 0.1, status=status)[0].cpu().numpy(), out)
    assert int(status.item()) == 0


@pytest.mark.parametrize("seqs", [150, 200, 260, 1030])
def test_decode_many_short_sequences_in_wide_tables(seqs):
    """More rows than SMs, tables of over 2048 tokens: splits by length, the list, and past the list's sequences."""
    g = np.random.default_rng(seqs)
    lens = g.integers(0, 6, seqs)
    lens[seqs // 2] = 700
    c = Case(seqs, lens, 1, 4, 64)
    c.table = np.concatenate([c.table, np.full((seqs, 40), -1, np.int32)], 1)
    out = _decode(c)
    c.check(out, 128 ** -0.5)
    assert np.array_equal(out, _decode(c)), "results depend on timing"


@pytest.mark.parametrize("softcap", [1e3, 1e5, 1e8, 1e20, 3e38])
@pytest.mark.parametrize("scale", [0.35, -0.35])
def test_decode_large_softcaps(softcap, scale):
    """Caps far above the scores, down to where the cap changes nothing.  Scores reach |s| < 24, and the
    capped one is within 2^-20 of its own size, so each p is within 2^-19 |s| more than without a cap:
    24 2^-19 on numerator and denominator add 10^-4 A to the bound."""
    c = Case(16, [1, 33, 257], 1, 4)
    out = _decode(c, softcap=softcap, scale=scale)
    for b in range(3):
        kk, vv = c.values(b)
        assert np.abs(np.einsum("hd,td->ht", c.q[b].astype(np.float64), kk[:, 0])).max() * abs(scale) < 24
        ref, a = kv_int4.attend(c.q[b], kk, vv, scale, 0, softcap)
        bound = (2.0 ** -10 * (1 + 2.0 ** -4) + 1e-4) * a + 2e-5 * np.abs(vv).max()
        assert (np.abs(out[b] - ref) <= bound).all()


@pytest.mark.parametrize("softcap", [0.01, 1.0, 15.0, 100.0])
def test_decode_softcap_on_both_sides_of_its_two_forms(softcap):
    """Scores from a thousandth of the cap to many times it; the flat softmax shows small errors."""
    c = Case(17, [400], 2, 4)
    for scale in (1e-4 * softcap, 0.02 * softcap, 2.0 * softcap):
        c.check(_decode(c, softcap=softcap, scale=scale), scale, 0, softcap)


def _f16_cache(seed, B, n, width):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    pages = B * width
    cache = PagedKVCache(num_pages=pages, page_size=16, num_kv_heads=2, head_dim=128,
                         block_table=np.arange(pages, dtype=np.int32).reshape(B, width))
    for p in (cache.k_pool, cache.v_pool):
        p.copy_(torch.randn(p.shape, generator=g, device="cuda"))
    return cache, torch.randn((B, 8, 128), generator=g, device="cuda").half(), torch.full((B,), n, dtype=torch.int32,
                                                                                          device="cuda")


def test_a_kept_workspace_serves_one_kind_of_cache():
    """int4 decodes keep their counters where the f16 and int8 decodes put partial sums: one workspace
    for both is refused, whichever came first."""
    c = Case(91, [3000, 2500], 2, 4)
    cache = c.cache()
    old, q, n = _f16_cache(1, 2, 3000, 188)
    size = max(ops.decode_workspace(x, 2, 8).numel() for x in (cache, old))
    for first in ("int4", "f16"):
        ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
        four = lambda: _decode(c, cache, ws=ws)
        half = lambda: ops.paged_decode(old, q, n, 0.1, ws=ws)
        a, b = (four, half) if first == "int4" else (half, four)
        a()
        with pytest.raises(ValueError):
            b()
        a()
    c.check(_decode(c, cache, ws=torch.zeros(size, dtype=torch.uint8, device="cuda")), 128 ** -0.5)


def test_f16_decodes_of_several_shapes_on_one_workspace():
    """Their counters lie behind partial sums whose size follows the shape: another shape clears them."""
    shapes = [_f16_cache(2, 4, 3000, 188), _f16_cache(3, 1, 5000, 313), _f16_cache(4, 9, 700, 44)]
    want = [ops.paged_decode(cache, q, n, 0.1).clone() for cache, q, n in shapes]
    ws = torch.zeros(max(ops.decode_workspace(cache, q.shape[0], 8).numel() for cache, q, n in shapes), dtype=torch.uint8,
                     device="cuda")
    for _ in range(2):
        for (cache, q, n), w in zip(shapes, want):
            for _ in range(2):
                out = torch.full_like(w, 7.0)
                ops.paged_decode(cache, q, n, 0.1, ws=ws, out=out)
                assert torch.equal(out, w)


def test_int4_decodes_of_several_shapes_on_one_workspace():
    cases = [Case(92, [3000, 2500], 2, 4), Case(93, [5000], 1, 8), Case(94, [700] * 9, 2, 2)]
    caches = [c.cache() for c in cases]
    want = [_decode(c, k) for c, k in zip(cases, caches)]
    ws = torch.zeros(max(ops.decode_workspace(k, len(c.lens), c.H).numel() for c, k in zip(cases, caches)),
                     dtype=torch.uint8, device="cuda")
    for _ in range(2):
        for c, k, w in zip(cases, caches, want):
            assert np.array_equal(_decode(c, k, ws=ws), w)


def test_a_decode_captured_on_a_given_stream_has_its_own_workspace(monkeypatch):
    """stream= names a stream that is being captured while the current one is not."""
    c = Case(72, [3000, 2500], 2, 4)
    cache, q, n = c.cache(), _t(c.q), _t(c.lens)
    main, side, idle = (torch.cuda.Stream() for _ in range(3))
    torch.cuda.synchronize()
    want = ops.paged_decode(cache, q, n, 0.1, stream=side)
    got = torch.empty_like(want)
    torch.cuda.synchronize()

    def kept(*_):
        raise AssertionError("the stream's workspace went into the graph")

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        side.wait_stream(main)
        with monkeypatch.context() as m:
            m.setattr(ops, "_kept_workspace", kept)
            with torch.cuda.stream(idle):
                ops.paged_decode(cache, q, n, 0.1, out=got, stream=side)
        main.wait_stream(side)
    for _ in range(3):
        got.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_a_stream_of_the_callers_own_has_no_kept_workspace():
    """A stream that torch did not make can be destroyed, and its handle be another stream's then."""
    c = Case(73, [3000, 2500], 2, 4)
    cache, q, n = c.cache(), _t(c.q), _t(c.lens)
    want = ops.paged_decode(cache, q, n, 0.1)
    made = torch.cuda.Stream()
    torch.cuda.synchronize()
    before = set(ops._DECODE_WS)
    handle = ctypes.c_void_p()
    assert torch.cuda.cudart().cudaStreamCreate(ctypes.addressof(handle)) == 0
    try:
        s = torch.cuda.ExternalStream(handle.value)
        outs = [ops.paged_decode(cache, q, n, 0.1, stream=s)]
        with torch.cuda.stream(s):
            outs.append(ops.paged_decode(cache, q, n, 0.1))
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
        assert set(ops._DECODE_WS) == before
        ops._DECODE_WS.pop((0, made.cuda_stream), None)
        out = ops.paged_decode(cache, q, n, 0.1, stream=made)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and (0, made.cuda_stream) in ops._DECODE_WS
    finally:
        assert torch.cuda.cudart().cudaStreamDestroy(handle.value) == 0


@pytest.mark.parametrize("vstd", [1e-6, 1e-5, 1e-4, 1e-2, 1.0, 30.0, 1000.0, 9000.0])
def test_decode_long_tails_at_every_magnitude_of_v(vstd):
    """Each warp walks one key of 2^14.4 times the weight of its other 15000, which carry 0.4 of the sum.
    s p is held in f16 over 17 powers of two below the largest key's, so a tail key's is rounded to 2^-11
    of itself; p is too (2^-10 of the sum together, as V has one sign), and V is what the cache holds."""
    n = 60000
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    pages = n // 16
    cache = PagedKVCache(num_pages=pages, page_size=16, num_kv_heads=1, head_dim=128,
                         block_table=np.arange(pages, dtype=np.int32)[None], kv_dtype="int4")
    q = torch.ones((1, 4, 128), device="cuda").half()
    k = torch.zeros((1, n, 1, 128), device="cuda").half()
    k[0, [0, 16, 32, 48]] = 1.0  # one block of each of a CTA's four warps
    v = (torch.randn((1, n, 1, 128), generator=g, device="cuda").abs() * vstd).clamp(max=65504.0).half()
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.paged_append(cache, k, v, zero)
    scale = 14.4 * np.log(2) / 128
    out = ops.paged_decode(cache, q, torch.full((1,), n, dtype=torch.int32, device="cuda"), scale, split_pages=pages)
    kk, vv = (x[0, :, 0].double() for x in ops.paged_read(cache, zero, n, dtype=torch.float32))
    p = torch.softmax((q[0].double() @ kk.T) * scale, -1)
    ref = p @ vv
    assert bool(((out[0].double() - ref).abs() <= 2.0 ** -9 * ref).all()), float(((out[0] - ref).abs() / ref).max())


def _ragged(n, *more):
    return [(7 * i * i) % 41 for i in range(n)] + list(more)


# Each way a launch is cut up: lengths, kv heads, heads per kv head, unused pages per table row, window
PLANS = {
    "splits by length": (_ragged(9, 1, 2, 15, 16, 17, 31, 32, 33, 65, 300, 700), 2, 4, 0, 37),
    "clusters by length": ([1, 2600, 17, 0, 300], 1, 5, 200, 2100),        # table of more than 256 blocks, few rows
    "pieces of one list": (_ragged(130, 2300, 150, 2049), 2, 4, 0, 2100),   # more than a 7th of the warps' rows
    "pieces, one head": (_ragged(256, 700, 2300), 1, 3, 0, 2250),
    "a CTA a row": (_ragged(40, 300, 1, 129), 4, 2, 0, 100),                # tables of at most 128 blocks
    "past the list": (_ragged(1028, 700, 40), 1, 1, 140, 2100),              # more than 1024 sequences
}


@pytest.mark.parametrize("rope,stable,windowed,softcap,bf16", [
    (False, False, False, 0.0, False), (True, True, False, 0.0, True), (True, False, True, 0.0, False),
    (False, True, True, 20.0, True)])
@pytest.mark.parametrize("plan", PLANS)
def test_decode_appends_in_every_plan(plan, rope, stable, windowed, softcap, bf16):
    lens, Hkv, group, wide, window = PLANS[plan]
    window = window if windowed else 0
    c = Case(len(lens), lens, Hkv, group)
    c.table = np.concatenate([c.table, np.full((len(lens), wide), -1, np.int32)], 1)
    B = len(lens)
    nk, nv = _rows(c.g, (B, Hkv, 128)), _rows(c.g, (B, Hkv, 128), 3.0)
    last = c.lens.astype(np.int64) - 1
    cis = rope_table(int(last.max()) + 1, 128, 10000.0)
    rk, q = (kv_int4.rotate(nk, last, cis), kv_int4.rotate(c.q, last, cis)) if rope else (nk, c.q)
    cache = c.cache()
    out = _decode(c, cache, new_k=_t(nk), new_v=_t(nv), freq_cis=_t(cis) if rope else None, inputs_stable=stable,
                  sliding_window=window, softcap=softcap, out_dtype=torch.bfloat16 if bf16 else torch.float32)
    k, v = c.k.copy(), c.v.copy()
    for b in range(B):
        k[b, last[b]], v[b, last[b]] = rk[b], nv[b]  # of an empty sequence: a row that nobody reads
    c.check(out, 128 ** -0.5, window, softcap, q=q, k=k, v=v, bf16=bf16)
    kv_int4.append(c.kp, c.vp, c.table, 16, rk[:, None], nv[:, None], last)
    assert np.array_equal(cache.k_pool.cpu().numpy(), c.kp), "the append wrote other K bytes"
    assert np.array_equal(cache.v_pool.cpu().numpy(), c.vp), "the append wrote other V bytes"


@pytest.mark.parametrize("plan", PLANS)
def test_decode_reports_bad_pages_and_lengths_in_every_plan(plan):
    """One sequence has pages outside the pool (their keys are left out), two have lengths outside the
    table; the others are not touched."""
    lens, Hkv, group, wide, _ = PLANS[plan]
    c = Case(len(lens), lens, Hkv, group)
    c.table = np.concatenate([c.table, np.full((len(lens), wide), -1, np.int32)], 1)
    b = int(np.argmax(c.lens))
    pages = -(-int(c.lens[b]) // 16)
    bad = np.arange(pages)[1::3]
    c.table[b, bad[::2]], c.table[b, bad[1::2]] = c.pages, -7
    short = [i for i in range(len(lens)) if 0 < lens[i] < 20][:2]
    given = c.lens.copy()
    given[short[0]], given[short[1]] = -3, 10 ** 6  # nothing; the row up to its end, which is unmapped
    status = ops.status_word()
    out = ops.paged_decode(c.cache(), _t(c.q), _t(given), 128 ** -0.5, status=status).cpu().numpy()
    assert int(status.item()) == DOE_DEVICE_ERR_PAGE | DOE_DEVICE_ERR_LENGTH
    assert not out[short[0]].any()
    keep = np.ones(int(c.lens[b]), bool)
    for p in bad:
        keep[16 * p:16 * p + 16] = False
    for i in range(len(lens)):
        if i == short[0]:
            continue
        kk, vv = c.values(i)
        if i == short[1]:  # the last page's unwritten rows are attended too: anything
            continue
        if i == b:
            kk, vv = kk[keep], vv[keep]
        ref, a = kv_int4.attend(c.q[i], kk, vv, 128 ** -0.5)
        bound = 2.0 ** -10 * (1 + 2.0 ** -4) * a + 2e-5 * (np.abs(vv).max() if len(vv) else 0.0)
        assert (np.abs(out[i] - ref) <= bound).all(), i


@pytest.mark.parametrize("kv_dtype,good,bad", [("f16", torch.float16, torch.bfloat16), ("int8", torch.int8, torch.float8_e4m3fn),
                                               ("int4", torch.uint8, torch.float8_e5m2)])
def test_pools_of_another_floating_type_are_refused(kv_dtype, good, bad):
    """Their elements have the size of the right ones, and would be read as those."""
    n = 1152 if kv_dtype == "int4" else 16 * 128
    pool = lambda dt: torch.zeros(n, dtype=dt, device="cuda")
    scale = lambda dt: torch.zeros(16, dtype=dt, device="cuda") if kv_dtype == "int8" else None
    make = lambda k, v, s: PagedKVCache.from_pools(k, v, page_size=16, num_kv_heads=1, head_dim=128, kv_dtype=kv_dtype,
                                                   block_table=_t(np.zeros((1, 1), np.int32)), k_scale=s, v_scale=s)
    assert make(pool(good), pool(good), scale(torch.float16)).num_pages == 1
    with pytest.raises(ValueError):
        make(pool(bad), pool(good), scale(torch.float16))
    with pytest.raises(ValueError):
        make(pool(good), pool(bad), scale(torch.float16))
    if kv_dtype == "int8":
        with pytest.raises(ValueError):
            make(pool(good), pool(good), scale(torch.bfloat16))
