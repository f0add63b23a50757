"""torch-facing wrappers of the operator surface (include/doe_cuda.h).

Each wrapper validates shapes / dtypes, passes raw device pointers and the
current torch stream to libdoe_cuda.so, and raises DoeError on a non-OK
status.  Nothing here computes on the host.
"""
from __future__ import annotations

import ctypes as C
from functools import lru_cache
from typing import NamedTuple

import numpy as np
import torch

from . import _abi as abi
from .kv import KV_DTYPES, PagedKVCache

_WS: dict[int, torch.Tensor] = {}


def workspace(nbytes: int, device=None) -> torch.Tensor:
    """A cached device scratch buffer of at least nbytes (grown on demand)."""
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    key = dev.index if dev.index is not None else torch.cuda.current_device()
    buf = _WS.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=dev)
        _WS[key] = buf
    return buf


def _stream_handle(stream, device) -> int:
    """The cudaStream_t of `stream`, or of the device's current stream (without building a
    torch.cuda.Stream, which costs more than the rest of a wrapper)."""
    if stream is not None:
        return stream.cuda_stream
    index = device.index if isinstance(device, torch.device) else None
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if index is None else index)


def _launch(ws_bytes: int = 0, status: torch.Tensor | None = None, stream=None, device=None) -> abi.Launch:
    ws = workspace(ws_bytes, device) if ws_bytes else None
    return abi.Launch(_stream_handle(stream, device), ws.data_ptr() if ws is not None else None,
                      ws.numel() if ws is not None else 0,
                      status.data_ptr() if status is not None else None)


def _need(t: torch.Tensor, dtype, name: str) -> None:
    if not t.is_cuda or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous CUDA {dtype} tensor")


def status_word(device=None) -> torch.Tensor:
    """A zeroed device int32 that kernels OR DOE_DEVICE_ERR_* bits into."""
    return torch.zeros(1, dtype=torch.int32, device=device or "cuda")


def attention_decode_f32(q, k_cache, v_cache, scale: float, out=None, status=None, stream=None):
    """attention-decode.wgsl: q [H,D], k/v [H,L,D] f32 -> [H,D]."""
    for t, n in ((q, "q"), (k_cache, "k_cache"), (v_cache, "v_cache")):
        _need(t, torch.float32, n)
    H, D = q.shape
    L = k_cache.shape[1]
    out = torch.empty_like(q) if out is None else out
    lib = abi.lib()
    ws = lib.doe_attention_decode_f32_workspace_bytes(H, D, L)
    l = _launch(ws, status, stream, q.device)
    abi.check("doe_attention_decode_f32", lib.doe_attention_decode_f32(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), H, D, L, float(scale),
        C.byref(l)))
    return out


def attention_online(u: dict, q, k, v, kv_len_buffer=None, page_table=None, out=None, status=None,
                     stream=None):
    """attention_head256_f16kv.wgsl semantics: q [query_len,H,D] f32, k/v [pos,Hkv,D] f16|f32."""
    _need(q, torch.float32, "q")
    kv_elem = 1 if k.dtype == torch.float32 else 0
    uni = abi.AttnUniforms(**{**u, "pad": 0})
    out = torch.zeros_like(q) if out is None else out
    l = _launch(0, status, stream, q.device)
    abi.check("doe_attention_online", abi.lib().doe_attention_online(
        C.byref(uni), q.data_ptr(), k.data_ptr(), v.data_ptr(), kv_elem, out.data_ptr(),
        kv_len_buffer.data_ptr() if kv_len_buffer is not None else None,
        page_table.data_ptr() if page_table is not None else None, C.byref(l)))
    return out


def attention_prefill_wgsl(q, k, v, scale: float, out=None, status=None, stream=None):
    """attention-prefill.wgsl: causal, [H,S,D] f32."""
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _need(t, torch.float32, n)
    H, S, D = q.shape
    out = torch.empty_like(q) if out is None else out
    l = _launch(0, status, stream, q.device)
    abi.check("doe_attention_prefill_wgsl_f32", abi.lib().doe_attention_prefill_wgsl_f32(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), S, D, H, float(scale), C.byref(l)))
    return out


def stitch(partials, out=None, stream=None):
    """[rows, shards, D+2] f32 partials -> [rows, D]."""
    _need(partials, torch.float32, "partials")
    rows, shards, w = partials.shape
    out = torch.empty((rows, w - 2), dtype=torch.float32, device=partials.device) if out is None else out
    l = _launch(0, None, stream, partials.device)
    abi.check("doe_attention_stitch_f32", abi.lib().doe_attention_stitch_f32(
        partials.data_ptr(), rows, shards, w - 2, out.data_ptr(), C.byref(l)))
    return out


@lru_cache(maxsize=256)
def _decode_need(B, H, split_pages, kv_dtype, num_pages, page_size, kv_heads, head_dim, max_pages, device) -> int:
    """doe_paged_decode_workspace_bytes, which depends on these sizes (and the device's SM count) alone."""
    kv = abi.PagedKV(1, 1, 1, 1, KV_DTYPES[kv_dtype], num_pages, page_size, kv_heads, head_dim, max_pages, 1)
    return int(abi.lib().doe_paged_decode_workspace_bytes(C.byref(kv), B, H, split_pages))


def paged_decode(cache: PagedKVCache, q, seq_lens, scale: float, new_k=None, new_v=None, out=None,
                 split_pages: int = 0, status=None, stream=None, freq_cis=None, sliding_window: int = 0,
                 softcap: float = 0.0, out_dtype=torch.float32, ws=None, inputs_stable: bool = False):
    """Batched GQA decode: q [B,H,D] f16, seq_lens [B] int32 -> out [B,H,D] f32.

    With new_k/new_v ([B,Hkv,D] f16) the new token is first written at
    position seq_lens[b] - 1 (quantised for int8 and int4 caches).  With freq_cis
    ([positions, D/2, 2] f32 RoPE table) the query and the new K row are
    rotated at position seq_lens[b] - 1 first (doe_paged_decode_rope).
    sliding_window > 0 keeps the last sliding_window keys and softcap > 0
    caps each scaled score as softcap * tanh(s / softcap) (doe_paged_decode_ex).
    out_dtype torch.bfloat16 writes a bf16 output (DOE_DECODE_OUT_BF16).
    `ws`: a workspace kept for paged decodes alone, zeroed when created
    (decode_workspace); its split counters then need no clearing per call
    (DOE_DECODE_COUNTERS_ZEROED).  One tensor serves int4 caches, of any shapes,
    or f16 and int8 ones (a call of another shape or type than the last one
    clears them), and never both; what a graph was captured with serves no other
    shape.  int4 caches keep one per stream of torch's by
    themselves (a captured graph gets its own).  inputs_stable: seq_lens, the block table and
    the pool rows (other than the appended ones) are final before the call is
    enqueued, so the first copies may start before the preceding kernel ends
    (DOE_DECODE_INPUTS_STABLE)."""
    _need(q, torch.float16, "q")
    _need(seq_lens, torch.int32, "seq_lens")
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("out_dtype must be float32 or bfloat16")
    B, H, D = q.shape
    if cache.kv_dtype == "int4":
        _rows_of(cache, B)
        if D != cache.head_dim or seq_lens.numel() != B:
            raise ValueError(f"q must be [B, H, {cache.head_dim}] and seq_lens [B]")
        if new_k is not None and new_v is not None:
            _need(new_k, torch.float16, "new_k")
            _need(new_v, torch.float16, "new_v")
            if not new_k.shape == new_v.shape == (B, cache.num_kv_heads, D):
                raise ValueError(f"new_k and new_v must be [{B}, {cache.num_kv_heads}, {D}]")
    out = torch.empty((B, H, D), dtype=out_dtype, device=q.device) if out is None else out
    _need(out, out_dtype, "out")
    flags = abi.DECODE_OUT_BF16 if out_dtype == torch.bfloat16 else 0
    if inputs_stable:
        flags |= abi.DECODE_INPUTS_STABLE
    kv = cache.struct()
    lib = abi.lib()
    need = _decode_need(B, H, split_pages, cache.kv_dtype, cache.num_pages, cache.page_size, cache.num_kv_heads,
                        cache.head_dim, cache.max_pages_per_seq, q.device.index)
    shared = ws is None and cache.kv_dtype != "int4"  # the workspace of all operators
    s = None if shared else _stream_handle(stream, q.device)
    given, kept = ws, None
    # a graph that is being captured holds a workspace of its own, cleared in every replay
    if ws is None and not shared and not _capturing(stream):
        kept = ws = _kept_workspace(need, q.device, s, stream)
    if given is not None:
        if given.numel() < need:
            raise ValueError(f"decode workspace of {need} bytes needed, {given.numel()} given")
        layout = "int4" if cache.kv_dtype == "int4" else (B * cache.num_kv_heads, need)
        last = getattr(given, "_decode_layout", layout)
        if (last == "int4") != (layout == "int4"):
            raise ValueError("a decode workspace serves int4 caches or f16 and int8 ones, not both")
    if kept is not None or (given is not None and last == layout):
        flags |= abi.DECODE_COUNTERS_ZEROED
    if shared:
        l = _launch(need, status, stream, q.device)
    else:
        if ws is None:
            with torch.cuda.stream(stream):
                ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        l = abi.Launch(s, ws.data_ptr(), ws.numel(), status.data_ptr() if status is not None else None)
    nk = new_k.data_ptr() if new_k is not None else None
    nv = new_v.data_ptr() if new_v is not None else None
    if sliding_window or softcap or flags:
        if freq_cis is not None:
            _need(freq_cis, torch.float32, "freq_cis")
        opts = abi.DecodeOptions(freq_cis.data_ptr() if freq_cis is not None else None,
                                 freq_cis.shape[0] if freq_cis is not None else 0, int(sliding_window),
                                 float(softcap), flags)
        abi.check("doe_paged_decode_ex", lib.doe_paged_decode_ex(
            C.byref(kv), B, H, q.data_ptr(), seq_lens.data_ptr(), nk, nv, float(scale), out.data_ptr(),
            split_pages, C.byref(opts), C.byref(l)))
    elif freq_cis is None:
        abi.check("doe_paged_decode", lib.doe_paged_decode(
            C.byref(kv), B, H, q.data_ptr(), seq_lens.data_ptr(), nk, nv, float(scale), out.data_ptr(),
            split_pages, C.byref(l)))
    else:
        _need(freq_cis, torch.float32, "freq_cis")
        abi.check("doe_paged_decode_rope", lib.doe_paged_decode_rope(
            C.byref(kv), B, H, q.data_ptr(), seq_lens.data_ptr(), nk, nv, float(scale), out.data_ptr(),
            split_pages, freq_cis.data_ptr(), freq_cis.shape[0], C.byref(l)))
    if given is not None:
        given._decode_layout = layout
    return out


def _capturing(stream) -> bool:
    """Whether `stream`, or the current one, is being captured into a graph."""
    if stream is None:
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.stream(stream):
        return torch.cuda.is_current_stream_capturing()


_DECODE_WS: dict[tuple[int, int], torch.Tensor] = {}


def _kept_workspace(nbytes: int, device, handle: int, stream) -> torch.Tensor | None:
    """The int4 decodes' own workspace of a stream: its counters stay zero from call to call, whatever
    the shapes (they come first), so no call clears them.  It lasts as long as the process, as torch's
    own streams do, of which there are a few dozen.  None for a stream that torch did not make: it can
    be destroyed with work pending, and another stream get its handle."""
    kept = _DECODE_WS.get((device.index, handle))
    if kept is not None and kept.numel() >= nbytes:
        return kept
    with torch.cuda.stream(stream):  # None: the current stream, which `handle` is then
        if handle and torch.cuda.current_stream(device).stream_id == handle:  # the id of a foreign stream
            return None
        kept = torch.zeros(max(nbytes, 1 << 22), dtype=torch.uint8, device=device)
    _DECODE_WS[device.index, handle] = kept
    return kept


def decode_workspace(cache: PagedKVCache, num_seqs: int, num_heads: int, split_pages: int = 0) -> torch.Tensor:
    """A zeroed workspace for paged decodes of this kind of cache alone (pass as paged_decode(ws=...))."""
    kv = cache.struct()
    need = int(abi.lib().doe_paged_decode_workspace_bytes(C.byref(kv), num_seqs, num_heads, split_pages))
    return torch.zeros(max(need, 256), dtype=torch.uint8, device=cache.k_pool.device)


def paged_append(cache: PagedKVCache, new_k, new_v, positions, status=None, stream=None, freq_cis=None):
    """Write new_k/new_v [B,T,Hkv,D] f16 at positions[b] + t (quantising int8 and int4 caches).

    With freq_cis ([positions, D/2, 2] f32 RoPE table) each K row is first
    rotated at its position (doe_paged_append_rope)."""
    _need(new_k, torch.float16, "new_k")
    _need(new_v, torch.float16, "new_v")
    _need(positions, torch.int32, "positions")
    B, T = new_k.shape[:2]
    if cache.kv_dtype == "int4":
        _rows_of(cache, B)
        if not new_k.shape == new_v.shape == (B, T, cache.num_kv_heads, cache.head_dim) or positions.numel() != B:
            raise ValueError(f"new_k and new_v must be [B, T, {cache.num_kv_heads}, {cache.head_dim}], positions [B]")
    kv = cache.struct()
    l = _launch(0, status, stream, new_k.device)
    if freq_cis is None:
        abi.check("doe_paged_append", abi.lib().doe_paged_append(
            C.byref(kv), B, T, new_k.data_ptr(), new_v.data_ptr(), positions.data_ptr(), C.byref(l)))
    else:
        _need(freq_cis, torch.float32, "freq_cis")
        abi.check("doe_paged_append_rope", abi.lib().doe_paged_append_rope(
            C.byref(kv), B, T, new_k.data_ptr(), new_v.data_ptr(), positions.data_ptr(), freq_cis.data_ptr(),
            freq_cis.shape[0], C.byref(l)))


def paged_gather(cache: PagedKVCache, seq: int, start: int, length: int, status=None, stream=None):
    """kv_read: tokens [start, start+length) of one sequence -> (k, v[, k_scale, v_scale])."""
    shape = (length, cache.num_kv_heads, cache.head_dim)
    k = torch.empty(shape, dtype=cache.k_pool.dtype, device=cache.k_pool.device)
    v = torch.empty_like(k)
    ks = vs = None
    if cache.kv_dtype == "int8":
        ks = torch.empty((length, cache.num_kv_heads), dtype=torch.float16, device=k.device)
        vs = torch.empty_like(ks)
    kv = cache.struct()
    l = _launch(0, status, stream, k.device)
    abi.check("doe_paged_gather", abi.lib().doe_paged_gather(
        C.byref(kv), seq, start, length, k.data_ptr(), v.data_ptr(),
        ks.data_ptr() if ks is not None else None, vs.data_ptr() if vs is not None else None,
        C.byref(l)))
    return (k, v) if ks is None else (k, v, ks, vs)


def paged_read(cache: PagedKVCache, positions, n_tokens: int, dtype=torch.float16, out=None, status=None, stream=None):
    """kv_read as values: tokens positions[b] .. + n_tokens of every sequence b (block-table
    row b) -> (k, v) [B, n_tokens, Hkv, D] of dtype (f16, bf16 or f32), for any cache type.

    Rows on unmapped pages are zeros (and set DOE_DEVICE_ERR_PAGE in `status`)."""
    _need(positions, torch.int32, "positions")
    if dtype not in _DTYPES:
        raise ValueError("dtype must be float16, bfloat16 or float32")
    B = _rows_of(cache, positions.numel())
    shape = (B, int(n_tokens), cache.num_kv_heads, cache.head_dim)
    if out is None:
        k = torch.empty(shape, dtype=dtype, device=positions.device)
        v = torch.empty_like(k)
    else:
        k, v = out
        for t, n in ((k, "out k"), (v, "out v")):
            _need(t, dtype, n)
            if tuple(t.shape) != shape:
                raise ValueError(f"{n} must be {shape}")
    kv = cache.struct()
    l = _launch(0, status, stream, positions.device)
    abi.check("doe_paged_read", abi.lib().doe_paged_read(
        C.byref(kv), B, shape[1], positions.data_ptr(), k.data_ptr(), v.data_ptr(), _DTYPES[dtype], C.byref(l)))
    return k, v


def _rows_of(cache: PagedKVCache, n: int) -> int:
    if n > cache.block_table.shape[0]:
        raise ValueError(f"{n} sequences, the block table has {cache.block_table.shape[0]} rows")
    return n


def paged_copy_pages(cache: PagedKVCache, pairs, stream=None) -> None:
    """Copies pages pairs[i][0] -> pairs[i][1] (K, V and scales) inside the cache.

    `pairs` [n, 2] is on the host (KvPool.make_writable, KvPool.compact); no
    page may be a target twice, or a target and a source."""
    p = np.ascontiguousarray(pairs, dtype=np.int32)
    if p.size and (p.ndim != 2 or p.shape[1] != 2):
        raise ValueError("pairs must be [n, 2]")
    kv = cache.struct()
    l = _launch(0, None, stream, cache.k_pool.device)
    abi.check("doe_paged_copy_pages", abi.lib().doe_paged_copy_pages(C.byref(kv), p.ctypes.data, p.size // 2, C.byref(l)))


class TokenLogprobs(NamedTuple):
    """token_logprobs' results; logprob is None without tokens, top_* are [rows, 0] for top_k 0."""

    logprob: torch.Tensor | None   # [rows] f32
    entropy: torch.Tensor          # [rows] f32
    top_ids: torch.Tensor          # [rows, top_k] int32
    top_logprobs: torch.Tensor     # [rows, top_k] f32


def token_logprobs(logits, tokens=None, top_k: int = 0, status=None, stream=None) -> TokenLogprobs:
    """Log probabilities of tokens [rows] int32 under logits [rows, vocab] (f32, f16 or bf16; rows
    may be strided), each row's entropy (natural logarithm) and its top_k <= 32 alternatives, ties
    to the lowest index (doe_token_logprobs)."""
    if not logits.is_cuda or logits.dtype not in _DTYPES or logits.ndim != 2 or logits.stride(1) != 1 \
            or (logits.shape[0] > 1 and logits.stride(0) < logits.shape[1]):
        raise ValueError("logits must be a CUDA f32, f16 or bf16 [rows, vocab] tensor with contiguous rows")
    rows, vocab = logits.shape
    if tokens is not None:
        _need(tokens, torch.int32, "tokens")
        if tokens.numel() != rows:
            raise ValueError(f"{rows} rows of logits, {tokens.numel()} tokens")
    dev = logits.device
    entropy = torch.empty(rows, dtype=torch.float32, device=dev)
    logprob = torch.empty_like(entropy) if tokens is not None else None
    top = torch.empty((rows, top_k), dtype=torch.float32, device=dev)
    ids = torch.empty_like(top, dtype=torch.int32)
    l = _launch(0, status, stream, dev)
    abi.check("doe_token_logprobs", abi.lib().doe_token_logprobs(
        logits.data_ptr(), _DTYPES[logits.dtype], rows, vocab, max(logits.stride(0), vocab),
        tokens.data_ptr() if tokens is not None else None, top_k, logprob.data_ptr() if tokens is not None else None,
        entropy.data_ptr(), ids.data_ptr() if top_k else None, top.data_ptr() if top_k else None, C.byref(l)))
    return TokenLogprobs(logprob, entropy, ids, top)


def kv_write_dense(k_proj, v_proj, k_cache, v_cache, positions, status=None, stream=None):
    """proj [heads, D], caches [heads, max_seq_len, D] (f16|f32), positions u32 [1|heads]."""
    heads, max_len, D = k_cache.shape
    eb = k_cache.element_size()
    l = _launch(0, status, stream, k_cache.device)
    abi.check("doe_kv_write_dense", abi.lib().doe_kv_write_dense(
        k_proj.data_ptr(), v_proj.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
        positions.data_ptr(), positions.numel(), heads, max_len, D, eb, C.byref(l)))


def kv_read_dense(k_cache, v_cache, read_start: int, read_len: int, status=None, stream=None):
    heads, max_len, D = k_cache.shape
    ko = torch.empty((heads, read_len, D), dtype=k_cache.dtype, device=k_cache.device)
    vo = torch.empty_like(ko)
    l = _launch(0, status, stream, k_cache.device)
    abi.check("doe_kv_read_dense", abi.lib().doe_kv_read_dense(
        k_cache.data_ptr(), v_cache.data_ptr(), ko.data_ptr(), vo.data_ptr(), heads, read_start,
        read_len, max_len, D, k_cache.element_size(), C.byref(l)))
    return ko, vo


def rope(qk, freq_cis, position_offset: int = 0, stream=None):
    """rope.wgsl in place on qk [S,H,D] f32."""
    _need(qk, torch.float32, "qk")
    S, H, D = qk.shape
    l = _launch(0, None, stream, qk.device)
    abi.check("doe_rope_f32", abi.lib().doe_rope_f32(
        qk.data_ptr(), freq_cis.data_ptr(), S, H, D, position_offset, C.byref(l)))
    return qk


def attention_prefill_f16(q, k, v, scale: float, causal: bool = True, cache: PagedKVCache | None = None,
                          cache_seq: int = 0, cache_start: int = 0, out=None, status=None, stream=None):
    """tcgen05 prefill: q [S,H,128], k/v [S,Hkv,128] f16 -> out [S,H,128] f32.

    With `cache`, the prompt's K/V rows are also written into the paged cache."""
    for t, n in ((q, "q"), (k, "k"), (v, "v")):
        _need(t, torch.float16, n)
    S, H, D = q.shape
    Hkv = k.shape[1]
    out = torch.empty((S, H, D), dtype=torch.float32, device=q.device) if out is None else out
    kv = cache.struct() if cache is not None else None
    l = _launch(0, status, stream, q.device)
    abi.check("doe_attention_prefill_f16", abi.lib().doe_attention_prefill_f16(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), S, H, Hkv, D, float(scale),
        1 if causal else 0, C.byref(kv) if kv is not None else None, cache_seq, cache_start,
        C.byref(l)))
    return out


_LINEAR_WS: dict[int, torch.Tensor] = {}


def linear_workspace(n_out: int, k: int, device=None) -> torch.Tensor:
    """The zero-initialised workspace doe_linear_bf16 keeps its tile counters in.

    Separate from `workspace()`: its counters must be zero before a call, and
    every call that completes without a timeout leaves them zero again."""
    dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
    key = dev.index if dev.index is not None else torch.cuda.current_device()
    need = int(abi.lib().doe_linear_workspace_bytes(n_out, k))
    buf = _LINEAR_WS.get(key)
    if buf is None or buf.numel() < need:
        buf = torch.zeros(need, dtype=torch.uint8, device=dev)
        _LINEAR_WS[key] = buf
    return buf


_DTYPES = {torch.bfloat16: abi.DTYPE_BF16, torch.float16: abi.DTYPE_F16, torch.float32: abi.DTYPE_F32}


def rmsnorm(x, gamma, eps: float, out=None, status=None, stream=None):
    """x [rows, cols] f32, gamma [cols] bf16 -> bf16 x / sqrt(mean(x^2) + eps) * gamma."""
    _need(x, torch.float32, "x")
    _need(gamma, torch.bfloat16, "gamma")
    rows, cols = x.shape
    out = torch.empty((rows, cols), dtype=torch.bfloat16, device=x.device) if out is None else out
    _need(out, torch.bfloat16, "out")
    l = _launch(0, status, stream, x.device)
    abi.check("doe_rmsnorm_bf16", abi.lib().doe_rmsnorm_bf16(
        x.data_ptr(), gamma.data_ptr(), float(eps), out.data_ptr(), rows, cols, C.byref(l)))
    return out


def ssq_buffer(cols: int, device=None) -> torch.Tensor:
    """The [cols / 32, 32] f32 sums of squares a norm-producing linear writes."""
    return torch.zeros((cols // 32, 32), dtype=torch.float32, device=device)


def linear(x, w, outs, *, swiglu: bool = False, residual=None, status=None, stream=None, ws=None,
           norm_out=None, norm_in=None):
    """doe_linear_bf16: x [batch, k] bf16 times w [n_out, k] bf16 transposed.

    `outs` is a list of 1-3 contiguous tensors of one dtype (bf16, f16 or f32),
    each [batch, width]; with swiglu=True a single [batch, n_out/2] output of
    silu(gate) * up (w packed in 128-row blocks: 64 gate rows, 64 up rows).
    `residual` ([batch, n_out] f32, f32 output) is added to the product.

    The RMSNorm between two products (doe_linear_bf16_norm): norm_out =
    (gamma [n_out] bf16, normed [batch, n_out] bf16, ssq (ssq_buffer(n_out)))
    makes this product (f32, one segment) also write bf16(y * gamma) and its
    per-32-column sums of squares; norm_in = (ssq, eps), with x such a normed
    output, scales each row of this product by 1 / sqrt(mean(h^2) + eps)."""
    _need(x, torch.bfloat16, "x")
    _need(w, torch.bfloat16, "w")
    batch, k = x.shape
    n_out = w.shape[0]
    if w.shape[1] != k:
        raise ValueError(f"w is {tuple(w.shape)}, x is {tuple(x.shape)}")
    if not 1 <= len(outs) <= 3:
        raise ValueError("1 to 3 output segments")
    dt = outs[0].dtype
    lo = abi.LinearOut()
    for i, o in enumerate(outs):
        _need(o, dt, f"outs[{i}]")
        lo.out[i] = o.data_ptr()
        lo.width[i] = o.shape[-1] if not swiglu else 0
    lo.dtype = _DTYPES[dt]
    lo.epilogue = abi.LINEAR_SWIGLU if swiglu else abi.LINEAR_STORE
    if residual is not None:
        _need(residual, torch.float32, "residual")
        lo.residual = residual.data_ptr()
    ws = linear_workspace(n_out, k, x.device) if ws is None else ws
    s = stream if stream is not None else torch.cuda.current_stream(x.device)
    l = abi.Launch(s.cuda_stream, ws.data_ptr(), ws.numel(), status.data_ptr() if status is not None else None)
    if norm_out is None and norm_in is None:
        abi.check("doe_linear_bf16", abi.lib().doe_linear_bf16(
            x.data_ptr(), w.data_ptr(), batch, n_out, k, C.byref(lo), C.byref(l)))
        return outs
    ln = abi.LinearNorm()
    if norm_out is not None:
        gamma, normed, ssq = norm_out
        _need(gamma, torch.bfloat16, "norm_out gamma")
        _need(normed, torch.bfloat16, "norm_out normed")
        _need(ssq, torch.float32, "norm_out ssq")
        if gamma.numel() != n_out or normed.shape != (batch, n_out) or ssq.numel() != n_out:
            raise ValueError("norm_out: gamma [n_out], normed [batch, n_out], ssq [n_out / 32, 32]")
        ln.gamma, ln.normed_out, ln.ssq_out = gamma.data_ptr(), normed.data_ptr(), ssq.data_ptr()
    if norm_in is not None:
        ssq, eps = norm_in
        _need(ssq, torch.float32, "norm_in ssq")
        if ssq.numel() != k:
            raise ValueError("norm_in: ssq [k / 32, 32]")
        ln.ssq_in, ln.eps = ssq.data_ptr(), float(eps)
    abi.check("doe_linear_bf16_norm", abi.lib().doe_linear_bf16_norm(
        x.data_ptr(), w.data_ptr(), batch, n_out, k, C.byref(lo), C.byref(ln), C.byref(l)))
    return outs
