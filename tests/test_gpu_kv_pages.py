"""GPU parity of page copies inside a paged cache: bytes equal, other pages untouched."""
from __future__ import annotations

import numpy as np
import pytest

from doe_b200 import ops
from doe_b200._abi import DoeError
from doe_b200.kv import KvPool, PagedKVCache

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def _filled(kv_dtype, pages, page, Hkv, D=128, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = PagedKVCache(num_pages=pages, page_size=page, num_kv_heads=Hkv, head_dim=D, block_table=np.zeros((1, 1)),
                     kv_dtype=kv_dtype)
    for t in (c.k_pool, c.v_pool, c.k_scale, c.v_scale):
        if t is not None:
            b = t.view(torch.uint8)
            b.copy_(torch.randint(0, 256, b.shape, generator=g, device="cuda", dtype=torch.uint8))
    return c


def _bytes(c):
    return [t.view(torch.uint8).reshape(c.num_pages, -1).cpu().numpy().copy()
            for t in (c.k_pool, c.v_pool, c.k_scale, c.v_scale) if t is not None]


@pytest.mark.parametrize("kv_dtype", ["f16", "int8", "int4"])
@pytest.mark.parametrize("page,Hkv", [(16, 1), (16, 8), (48, 3), (64, 8), (128, 2)])
@pytest.mark.parametrize("n", [1, 7, 60, 61])
def test_copies(kv_dtype, page, Hkv, n):
    c = _filled(kv_dtype, 150, page, Hkv)
    order = np.random.default_rng(n).permutation(150).astype(np.int32)
    pairs = np.stack([order[:n], order[n:2 * n]], 1)
    pairs[n // 2:, 0] = pairs[0, 0]  # one source for several targets
    want = _bytes(c)
    ops.paged_copy_pages(c, pairs)
    for w in want:
        w[pairs[:, 1]] = w[pairs[:, 0]]
    for a, w in zip(_bytes(c), want):
        assert np.array_equal(a, w)


def test_lists_longer_than_one_launch():
    c = _filled("int4", 9001, 16, 1)
    order = np.random.default_rng(0).permutation(9001).astype(np.int32)
    pairs = np.stack([order[:4500], order[4501:]], 1)
    want = _bytes(c)
    ops.paged_copy_pages(c, pairs)
    for a, w in zip(_bytes(c), want):
        w[pairs[:, 1]] = w[pairs[:, 0]]
        assert np.array_equal(a, w)


def test_empty_list_and_refusals():
    c = _filled("f16", 4, 16, 1)
    want = _bytes(c)
    ops.paged_copy_pages(c, np.empty((0, 2), np.int32))
    ops.paged_copy_pages(c, [])
    for bad in ([[0, 4]], [[-1, 1]], [[1, 1]], [[0, 2], [1, 2]], [[0, 1], [1, 2]]):
        with pytest.raises(DoeError):
            ops.paged_copy_pages(c, bad)
    with pytest.raises(ValueError):
        ops.paged_copy_pages(c, [[1, 2, 3]])
    torch.cuda.synchronize()
    assert all(np.array_equal(a, w) for a, w in zip(_bytes(c), want))


@pytest.mark.parametrize("kv_dtype", ["f16", "int4"])
def test_forked_sequences_diverge_without_touching_each_other(kv_dtype):
    """Fork, write one token each into the shared last page, compact: every sequence reads its own rows."""
    g = np.random.default_rng(1)
    pool = KvPool(64, 16, 6, 8)
    cache = PagedKVCache(num_pages=64, page_size=16, num_kv_heads=2, head_dim=128, block_table=pool.block_table(),
                         kv_dtype=kv_dtype)
    pool.reserve(5, 100)  # holes below the pages that stay
    prompt = 40
    pool.reserve(0, prompt)
    cache.set_block_table(pool.block_table())
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    k = g.standard_normal((1, prompt, 2, 128)).astype(np.float16)
    ops.paged_append(cache, t(k), t(k + 1), t(np.zeros(1, np.int32)))
    for s in (1, 2, 3):
        pool.fork(0, s, prompt)
    assert pool.free_pages() == 64 - 7 - 3
    pairs = np.concatenate([pool.make_writable(s, prompt, 1) for s in range(4)])
    assert len(pairs) == 3  # the last one keeps the page
    for s in range(4):
        pool.reserve(s, prompt + 1)
    ops.paged_copy_pages(cache, pairs)
    cache.set_block_table(pool.block_table())
    new = g.standard_normal((4, 1, 2, 128)).astype(np.float16)
    ops.paged_append(cache, t(new), t(new + 1), t(np.full(4, prompt, np.int32)))
    before = [x.cpu() for x in ops.paged_read(cache, t(np.zeros(4, np.int32)), prompt + 1)]
    for x in before:
        assert torch.equal(x[0, :prompt], x[3, :prompt]) and not torch.equal(x[0, prompt], x[3, prompt])
    if kv_dtype == "f16":
        assert torch.equal(before[0][2, prompt], torch.from_numpy(new[2, 0]))
    pool.release(5)
    pool.release(1)
    moves = pool.compact()
    assert len(moves)
    ops.paged_copy_pages(cache, moves)
    table = pool.block_table()
    assert table.max() < 64 - pool.free_pages()
    cache.set_block_table(table)
    after = ops.paged_read(cache, t(np.zeros(4, np.int32)), prompt + 1)
    for x, y in zip(before, after):
        for s in (0, 2, 3):
            assert torch.equal(x[s], y[s].cpu())
    pool.close()
