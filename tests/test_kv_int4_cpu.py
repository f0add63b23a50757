"""4-bit KV cache, page pool sharing and token log probabilities on the CPU: the
restated block layout against itself and the documented layout, the page pool
against a plain model, and the argument checks of the new entry points."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from doe_b200 import _abi as abi
from doe_b200.kv import KvPool
from oracle import kv_int4

FAKE = C.c_void_p(0x100000)  # never dereferenced


def test_restated_blocks_round_trip():
    g = np.random.default_rng(0)
    x = g.standard_normal((40, 2, 128)).astype(np.float16)
    x[3] = 0
    x[5, 0, :32] = 6e-8  # a subnormal scale that rounds to zero
    x[6, 1, 40] = 65504
    s, n = kv_int4.quantize(x)
    assert n.min() >= 1 and n.max() <= 15
    want = kv_int4.values(s, n)
    # error: half a step of the scale, the clamp where the f16 scale was rounded down
    step = np.repeat(s.astype(np.float64), 32, -1)
    assert (np.abs(want - x.astype(np.float64)) <= step * (0.5 + 7 * 2.0 ** -10) + 1e-7).all()
    table = np.array([[2, 0, 1]], np.int32)
    for is_v in (False, True):
        pool = np.zeros((3, 2, 1, 1152), np.uint8)
        for t in range(40):
            for h in range(2):
                kv_int4.put(pool, is_v, int(table[0, t // 16]), h, t % 16, s[t, h], n[t, h])
        assert np.array_equal(kv_int4.rows(pool, is_v, table[0], 16, 40), want)


def test_exact_halves_round_to_even():
    x = np.zeros((1, 128), np.float16)
    x[0, :7] = [7, 0.5, 1.5, 2.5, -0.5, -1.5, 6.5]  # scale 1
    _, n = kv_int4.quantize(x)
    assert n[0, :7].tolist() == [15, 8, 10, 10, 8, 6, 14]


class Model:
    """The page pool's contract, restated: rows of page ids, a page free when no row holds it."""

    def __init__(self, pages, page, seqs, width):
        self.pages, self.page, self.width = pages, page, width
        self.rows = [[] for _ in range(seqs)]

    def live(self):
        return {p for r in self.rows for p in r}


def _check(pool: KvPool, m: Model):
    bt = pool.block_table()
    rows = [[int(p) for p in r if p >= 0] for r in bt]
    assert [len(r) for r in rows] == [len(r) for r in m.rows]
    # the same sharing: equal pages in the model are equal pages in the pool and the other way round
    a = {}
    for r, q in zip(rows, m.rows):
        for p, v in zip(r, q):
            assert a.setdefault(v, p) == p
    assert len(set(a.values())) == len(a)
    assert pool.free_pages() == m.pages - len(a)
    for v, p in a.items():
        assert pool.page_refs(p) == sum(q.count(v) for q in m.rows)


@pytest.mark.parametrize("seed", range(6))
def test_page_pool_against_a_model(seed):
    g = np.random.default_rng(seed)
    pages, page, seqs, width = 24, 16, 6, 9
    pool, m = KvPool(pages, page, seqs, width), Model(pages, page, seqs, width)
    fresh = iter(range(10 ** 6))
    held = {}  # page -> contents, to check that the copy lists keep every sequence's data

    def contents():
        return [[held.get(int(p)) for p in r if p >= 0] for r in pool.block_table()]

    for _ in range(300):
        op, s, t = g.integers(0, 6), int(g.integers(0, seqs)), int(g.integers(0, seqs))
        before = contents()
        if op == 0:
            want = int(g.integers(0, width * page + 20))
            need = -(-want // page)
            extra = need - len(m.rows[s])
            if need > width or extra > pages - len(m.live()):
                with pytest.raises(abi.DoeError) as e:
                    pool.reserve(s, want)
                assert e.value.rc == abi.DOE_OUT_OF_RANGE and contents() == before
            else:
                pool.reserve(s, want)
                m.rows[s] += [next(fresh) for _ in range(max(0, extra))]
                for p in pool.block_table()[s]:
                    if p >= 0 and int(p) not in held:
                        held[int(p)] = object()
        elif op == 1:
            pool.release(s)
            m.rows[s] = []
        elif op == 2:
            keep = int(g.integers(0, width * page))
            pool.truncate(s, keep)
            m.rows[s] = m.rows[s][:-(-keep // page)]
        elif op == 3:
            tokens = int(g.integers(0, width * page))
            n = -(-tokens // page)
            if s == t or m.rows[t] or n > len(m.rows[s]):
                with pytest.raises(abi.DoeError):
                    pool.fork(s, t, tokens)
                assert contents() == before
            else:
                pool.fork(s, t, tokens)
                m.rows[t] = m.rows[s][:n]
                assert contents()[t] == before[s][:n]
        elif op == 4:
            first, count = int(g.integers(0, width * page)), int(g.integers(0, 40))
            p0, p1 = first // page, -(-(first + count) // page)
            if count and p1 > len(m.rows[s]):
                with pytest.raises(abi.DoeError):
                    pool.make_writable(s, first, count)
                assert contents() == before
                continue
            shared = [i for i in range(p0, p1) if count and sum(r.count(m.rows[s][i]) for r in m.rows) > 1]
            if len(shared) > pages - len(m.live()):
                with pytest.raises(abi.DoeError):
                    pool.make_writable(s, first, count)
                assert contents() == before
                continue
            pairs = pool.make_writable(s, first, count)
            assert len(pairs) == len(shared)
            for a, b in pairs.tolist():
                held[b] = held[a]
            for i in shared:
                m.rows[s][i] = next(fresh)
            assert contents() == before
        else:
            pairs = pool.compact()
            src, dst = set(pairs[:, 0].tolist()), set(pairs[:, 1].tolist())
            assert len(src) == len(dst) == len(pairs) and not src & dst
            for a, b in pairs.tolist():
                held[b] = held[a]
            assert contents() == before
            used = {int(p) for r in pool.block_table() for p in r if p >= 0}
            assert used == set(range(len(m.live())))
        live = {int(p) for r in pool.block_table() for p in r if p >= 0}
        held = {p: v for p, v in held.items() if p in live}
        _check(pool, m)
    pool.close()


def test_page_pool_refusals():
    pool = KvPool(4, 16, 3, 4)
    lib = abi.lib()
    n, v = C.c_uint32(), C.c_uint32()
    pool.reserve(0, 40)
    pool.fork(0, 1, 40)
    pairs = (C.c_int32 * 8)()
    # a list that is too small changes nothing
    assert lib.doe_kv_pool_make_writable(pool._h, 1, 0, 40, pairs, 2, C.byref(n)) == abi.DOE_OUT_OF_RANGE  # 1 free page
    assert lib.doe_kv_pool_make_writable(pool._h, 1, 0, 16, None, 0, C.byref(n)) == abi.DOE_INVALID_ARGUMENT
    assert lib.doe_kv_pool_make_writable(pool._h, 1, 0, 16, None, 3, C.byref(n)) == abi.DOE_INVALID_ARGUMENT
    assert lib.doe_kv_pool_make_writable(pool._h, 9, 0, 16, pairs, 4, C.byref(n)) == abi.DOE_OUT_OF_RANGE
    assert pool.free_pages() == 1 and n.value == 0
    assert len(pool.make_writable(1, 3, 0)) == 0
    assert pool.make_writable(1, 2 ** 32 - 1, 0).shape == (0, 2)
    with pytest.raises(abi.DoeError):
        pool.make_writable(1, 2 ** 32 - 1, 2)
    assert lib.doe_kv_pool_fork(None, 0, 1, 0) == abi.DOE_INVALID_ARGUMENT
    assert lib.doe_kv_pool_compact(pool._h, None, 1, C.byref(n)) == abi.DOE_INVALID_ARGUMENT
    assert lib.doe_kv_pool_page_refs(pool._h, 4, C.byref(v)) == abi.DOE_OUT_OF_RANGE
    assert lib.doe_kv_pool_truncate(pool._h, 3, 0) == abi.DOE_OUT_OF_RANGE
    pool.close()


def _kv(dtype=abi.DOE_KV_INT4, page=16, heads=8, dim=128, pool=FAKE, pages=10):
    return abi.PagedKV(pool, pool, None, None, dtype, pages, page, heads, dim, 4, FAKE)


def test_int4_argument_checks_precede_any_launch():
    lib = abi.lib()
    odd = C.c_void_p(0x100008)
    ok = _kv()
    assert lib.doe_paged_decode(C.byref(_kv(dim=64)), 1, 8, FAKE, FAKE, None, None, 1.0, FAKE, 0, None) == abi.DOE_UNSUPPORTED
    assert lib.doe_paged_append(C.byref(_kv(dim=256)), 1, 1, FAKE, FAKE, FAKE, None) == abi.DOE_UNSUPPORTED
    assert lib.doe_paged_append(C.byref(_kv(dtype=3)), 1, 1, FAKE, FAKE, FAKE, None) == abi.DOE_INVALID_ARGUMENT
    assert lib.doe_paged_append(C.byref(_kv(page=24)), 1, 1, FAKE, FAKE, FAKE, None) == abi.DOE_INVALID_ARGUMENT
    assert lib.doe_paged_append(C.byref(ok), 1, 1, odd, FAKE, FAKE, None) == abi.DOE_INVALID_ARGUMENT
    assert lib.doe_paged_append(C.byref(ok), 1, 2 ** 31, FAKE, FAKE, FAKE, None) == abi.DOE_INVALID_ARGUMENT
    assert lib.doe_paged_append(C.byref(ok), 65536, 1, FAKE, FAKE, FAKE, None) == abi.DOE_INVALID_ARGUMENT
    # nine heads per kv head; no workspace; a misaligned query
    assert lib.doe_paged_decode(C.byref(ok), 1, 72, FAKE, FAKE, None, None, 1.0, FAKE, 0, None) == abi.DOE_UNSUPPORTED
    assert "heads per kv head" in abi.op_error()
    assert lib.doe_paged_decode(C.byref(ok), 1, 8, FAKE, FAKE, None, None, 1.0, FAKE, 0, None) == abi.DOE_INVALID_ARGUMENT
    assert "workspace" in abi.op_error()
    l = abi.Launch(None, FAKE, 1 << 30, None)
    assert lib.doe_paged_decode(C.byref(ok), 1, 8, odd, FAKE, None, None, 1.0, FAKE, 0, C.byref(l)) == abi.DOE_INVALID_ARGUMENT
    # codes are not copied out row by row
    assert lib.doe_paged_gather(C.byref(ok), 0, 0, 1, FAKE, FAKE, None, None, None) == abi.DOE_UNSUPPORTED
    assert "doe_paged_read" in abi.op_error()
    # an int4 cache does not take the f16 prefill's fused write
    assert lib.doe_attention_prefill_f16(FAKE, FAKE, FAKE, FAKE, 16, 8, 8, 128, 1.0, 1, C.byref(ok), 0, 0, None) == \
        abi.DOE_INVALID_ARGUMENT


def test_read_and_copy_argument_checks():
    lib = abi.lib()
    odd = C.c_void_p(0x100008)
    ok = _kv()
    assert lib.doe_paged_read(C.byref(ok), 1, 1, None, FAKE, FAKE, 1, None) == abi.DOE_INVALID_ARGUMENT
    assert lib.doe_paged_read(C.byref(ok), 1, 1, FAKE, FAKE, FAKE, 3, None) == abi.DOE_INVALID_ARGUMENT
    assert lib.doe_paged_read(C.byref(ok), 1, 1, FAKE, odd, FAKE, 1, None) == abi.DOE_INVALID_ARGUMENT
    assert lib.doe_paged_read(C.byref(_kv(dtype=0, dim=12)), 1, 1, FAKE, FAKE, FAKE, 1, None) == abi.DOE_UNSUPPORTED
    assert lib.doe_paged_read(C.byref(ok), 0, 1, FAKE, FAKE, FAKE, 1, None) == abi.DOE_OK

    def copy(*pairs, kv=ok):
        flat = [p for q in pairs for p in q]
        return lib.doe_paged_copy_pages(C.byref(kv), (C.c_int32 * len(flat))(*flat), len(pairs), None)

    assert lib.doe_paged_copy_pages(C.byref(ok), None, 0, None) == abi.DOE_OK
    assert lib.doe_paged_copy_pages(C.byref(ok), None, 1, None) == abi.DOE_INVALID_ARGUMENT
    assert copy((0, 10)) == abi.DOE_OUT_OF_RANGE
    assert copy((-1, 3)) == abi.DOE_OUT_OF_RANGE
    assert copy((0, 0)) == abi.DOE_INVALID_ARGUMENT            # onto itself
    assert copy((0, 2), (1, 2)) == abi.DOE_INVALID_ARGUMENT    # one target twice
    assert copy((0, 2), (2, 3)) == abi.DOE_INVALID_ARGUMENT    # a target that is a source
    assert copy((2, 3), (0, 2)) == abi.DOE_INVALID_ARGUMENT
    assert copy((0, 1), kv=_kv(pool=odd)) == abi.DOE_INVALID_ARGUMENT
    assert copy((0, 1), (2, 3), (4, 5), kv=_kv(pages=2)) == abi.DOE_INVALID_ARGUMENT


def test_logprob_argument_checks():
    f = abi.lib().doe_token_logprobs

    def call(dtype=2, rows=1, vocab=10, stride=10, tokens=FAKE, k=1, lp=FAKE, ids=FAKE, top=FAKE, x=FAKE):
        return f(x, dtype, rows, vocab, stride, tokens, k, lp, FAKE, ids, top, None)

    assert call(rows=0) == abi.DOE_OK
    bad = [dict(dtype=3), dict(vocab=0), dict(stride=9), dict(k=33), dict(x=None), dict(tokens=None), dict(lp=None),
           dict(ids=None), dict(top=None), dict(k=0), dict(x=C.c_void_p(0x100002)), dict(dtype=1, x=C.c_void_p(0x100001)),
           dict(vocab=2 ** 31, stride=2 ** 31), dict(rows=2 ** 40)]
    for kw in bad:
        assert call(**kw) == abi.DOE_INVALID_ARGUMENT, kw
