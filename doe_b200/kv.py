"""KV-cache manager: the host page pool and the device-resident paged cache.

`KvPool` wraps the C pool in libdoe_cuda.so (physical page free list plus
per-sequence block-table rows).  `PagedKVCache` owns the device pools in the
layout the kernels read -- [num_pages * page_size, num_kv_heads, head_dim]
f16 or int8, int8 scales [num_pages, num_kv_heads, page_size] f16; int4 pools
[num_pages, num_kv_heads, page_size / 16, 1152] bytes (codes and scales of 16
tokens of one kv head) -- and a device copy of the block table.  This is the per-sequence generalisation of
the reference's single page_table binding
(attention_head256_f16kv.wgsl:38, get_kv_pos :51-63).
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _abi as abi


class KvPool:
    """Host page allocator (doe_kv_pool_*)."""

    def __init__(self, num_pages: int, page_size: int, max_seqs: int, max_pages_per_seq: int):
        self._lib = abi.lib()
        h = C.c_void_p()
        abi.check("doe_kv_pool_create",
                  self._lib.doe_kv_pool_create(num_pages, page_size, max_seqs, max_pages_per_seq,
                                               C.byref(h)))
        self._h = h
        self.num_pages, self.page_size = num_pages, page_size
        self.max_seqs, self.max_pages_per_seq = max_seqs, max_pages_per_seq

    def close(self) -> None:
        if self._h:
            self._lib.doe_kv_pool_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def reserve(self, seq: int, tokens: int) -> None:
        abi.check("doe_kv_pool_reserve", self._lib.doe_kv_pool_reserve(self._h, seq, tokens))

    def fork(self, src: int, dst: int, tokens: int) -> None:
        """Sequence dst (holding no page) shares the pages of src's first `tokens` tokens."""
        abi.check("doe_kv_pool_fork", self._lib.doe_kv_pool_fork(self._h, src, dst, tokens))

    def make_writable(self, seq: int, first_token: int, tokens: int) -> np.ndarray:
        """Gives seq pages of its own under tokens [first_token, + tokens): the (old, new)
        pages to copy before they are written, [n, 2] int32 (ops.paged_copy_pages)."""
        n = C.c_uint32()
        pairs = np.empty((tokens // self.page_size + 2, 2), np.int32)
        abi.check("doe_kv_pool_make_writable", self._lib.doe_kv_pool_make_writable(
            self._h, seq, first_token, tokens, pairs.ctypes.data, len(pairs), C.byref(n)))
        return pairs[:n.value]

    def truncate(self, seq: int, tokens: int) -> None:
        """Gives back the pages of seq past its first `tokens` tokens."""
        abi.check("doe_kv_pool_truncate", self._lib.doe_kv_pool_truncate(self._h, seq, tokens))

    def compact(self) -> np.ndarray:
        """Moves the live pages into the lowest ids: the (old, new) pages to copy, [n, 2] int32."""
        n = C.c_uint32()
        pairs = np.empty((self.num_pages, 2), np.int32)
        abi.check("doe_kv_pool_compact", self._lib.doe_kv_pool_compact(
            self._h, pairs.ctypes.data, len(pairs), C.byref(n)))
        return pairs[:n.value]

    def page_refs(self, page: int) -> int:
        """Sequences that hold `page` (0: free)."""
        v = C.c_uint32()
        abi.check("doe_kv_pool_page_refs", self._lib.doe_kv_pool_page_refs(self._h, page, C.byref(v)))
        return v.value

    def release(self, seq: int) -> None:
        abi.check("doe_kv_pool_release", self._lib.doe_kv_pool_release(self._h, seq))

    def free_pages(self) -> int:
        v = C.c_uint32()
        abi.check("doe_kv_pool_free_pages", self._lib.doe_kv_pool_free_pages(self._h, C.byref(v)))
        return v.value

    def seq_pages(self, seq: int) -> int:
        v = C.c_uint32()
        abi.check("doe_kv_pool_seq_pages", self._lib.doe_kv_pool_seq_pages(self._h, seq, C.byref(v)))
        return v.value

    def block_table(self) -> np.ndarray:
        out = np.empty((self.max_seqs, self.max_pages_per_seq), np.int32)
        abi.check("doe_kv_pool_block_table",
                  self._lib.doe_kv_pool_block_table(self._h, out.ctypes.data, out.size))
        return out


KV_DTYPES = {"f16": abi.DOE_KV_F16, "int8": abi.DOE_KV_INT8, "int4": abi.DOE_KV_INT4}


def _other_float(t) -> bool:
    """Of a floating type whose bytes the kernels would read as something else (integers may hold raw bytes)."""
    return t.dtype.is_floating_point and str(t.dtype) != "torch.float16"


class PagedKVCache:
    """Device pools + block table for the paged kernels (torch tensors on one GPU)."""

    def __init__(self, *, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 block_table, kv_dtype: str = "f16", device="cuda"):
        import torch

        if kv_dtype not in KV_DTYPES:
            raise ValueError("kv_dtype must be 'f16', 'int8' or 'int4'")
        if kv_dtype == "int4" and (head_dim != 128 or page_size % 16):
            raise ValueError("int4 pools need head_dim 128 and a page_size that is a multiple of 16")
        self.num_pages, self.page_size = num_pages, page_size
        self.num_kv_heads, self.head_dim = num_kv_heads, head_dim
        self.kv_dtype = kv_dtype
        if kv_dtype == "int4":
            shape = (num_pages, num_kv_heads, page_size // 16, abi.KV_INT4_BLOCK_BYTES)
            self.k_pool = torch.zeros(shape, dtype=torch.uint8, device=device)
        else:
            tdt = torch.float16 if kv_dtype == "f16" else torch.int8
            self.k_pool = torch.zeros((num_pages * page_size, num_kv_heads, head_dim), dtype=tdt, device=device)
        self.v_pool = torch.zeros_like(self.k_pool)
        if kv_dtype == "int8":
            self.k_scale = torch.zeros((num_pages, num_kv_heads, page_size), dtype=torch.float16,
                                       device=device)
            self.v_scale = torch.zeros_like(self.k_scale)
        else:
            self.k_scale = self.v_scale = None
        self.set_block_table(block_table)

    @classmethod
    def from_pools(cls, k_pool, v_pool, *, page_size: int, num_kv_heads: int, head_dim: int, block_table,
                   kv_dtype: str = "f16", k_scale=None, v_scale=None) -> "PagedKVCache":
        """A cache over pools (and int8 scales) that the caller holds, in the layouts above, and a
        block table on the pools' device ([sequences, pages] int32, used as it is)."""
        self = cls.__new__(cls)
        if kv_dtype not in KV_DTYPES:
            raise ValueError("kv_dtype must be 'f16', 'int8' or 'int4'")
        if kv_dtype == "int4" and (head_dim != 128 or page_size % 16):
            raise ValueError("int4 pools need head_dim 128 and a page_size that is a multiple of 16")
        if kv_dtype == "int8" and (k_scale is None or v_scale is None):
            raise ValueError("int8 pools need k_scale and v_scale")
        itemsize = {"f16": 2, "int8": 1, "int4": 1}[kv_dtype]
        row = num_kv_heads * (page_size // 16 * abi.KV_INT4_BLOCK_BYTES if kv_dtype == "int4"
                              else page_size * head_dim)
        if row <= 0 or k_pool.numel() % row or k_pool.numel() != v_pool.numel():
            raise ValueError("k_pool and v_pool must hold the same whole number of pages")
        for p in (k_pool, v_pool):
            if not p.is_cuda or not p.is_contiguous() or p.element_size() != itemsize or _other_float(p):
                raise ValueError(f"pools must be contiguous CUDA tensors of {kv_dtype} ({itemsize}-byte) elements")
        self.num_pages, self.page_size = k_pool.numel() // row, page_size
        if kv_dtype == "int8":
            for t in (k_scale, v_scale):
                if (not t.is_cuda or not t.is_contiguous() or t.element_size() != 2 or _other_float(t)
                        or t.numel() != self.num_pages * num_kv_heads * page_size):
                    raise ValueError("int8 scales must be contiguous CUDA f16 [pages, kv heads, page_size]")
        if not block_table.is_cuda or not block_table.is_contiguous() or block_table.ndim != 2 \
                or block_table.dtype.itemsize != 4 or block_table.dtype.is_floating_point:
            raise ValueError("block_table must be a contiguous 2-D CUDA int32 tensor")
        dev = k_pool.get_device()
        if not dev == v_pool.get_device() == block_table.get_device() or (
                kv_dtype == "int8" and not dev == k_scale.get_device() == v_scale.get_device()):
            raise ValueError("pools, scales and block_table must be on one device")
        self.num_kv_heads, self.head_dim, self.kv_dtype = num_kv_heads, head_dim, kv_dtype
        self.k_pool, self.v_pool, self.k_scale, self.v_scale = k_pool, v_pool, k_scale, v_scale
        self.block_table, self.max_pages_per_seq = block_table, block_table.shape[1]
        return self

    def set_block_table(self, block_table) -> None:
        import torch

        bt = torch.as_tensor(np.ascontiguousarray(block_table, dtype=np.int32))
        self.block_table = bt.to(self.k_pool.device)
        self.max_pages_per_seq = int(bt.shape[1])

    def struct(self) -> abi.PagedKV:
        return abi.PagedKV(
            self.k_pool.data_ptr(), self.v_pool.data_ptr(),
            self.k_scale.data_ptr() if self.k_scale is not None else None,
            self.v_scale.data_ptr() if self.v_scale is not None else None,
            KV_DTYPES[self.kv_dtype],
            self.num_pages, self.page_size, self.num_kv_heads, self.head_dim,
            self.max_pages_per_seq, self.block_table.data_ptr())

    def nbytes(self) -> int:
        n = self.k_pool.numel() * self.k_pool.element_size() * 2
        if self.k_scale is not None:
            n += self.k_scale.numel() * 2 * 2
        return n
