// kv_int4.cu -- writes into and reads out of the 4-bit paged KV cache.
//
//   append : f16 rows [B, T, Hkv, 128], K optionally rotated (rope.wgsl:12-35),
//            quantised into the blocks of int4.cuh
//   read   : value rows of any cache type (f16, int8, int4) as f16, bf16 or f32
//
// Copies with a little arithmetic: 512 bytes of f16 K and V against 144 bytes of
// blocks per (token, kv head).  Writing 32 x 512 tokens of 8 kv heads and reading them
// back takes 33.4 us for 172 MB (5.1 TB/s, 0.79 of the measured copy rate); the write
// alone is near 20, bound by issue slots (79 instructions for a token's K or V of a
// head, half of the cycles) and by how many loads 20 warps an SM keep in flight, the
// read near 14, bound by HBM writes and the two loads before its own.  32 tokens
// written and read back take 6.5 us: two launches.
#include <type_traits>

#include "int4.cuh"

namespace doe {

// Positions are below 2^32 (an int32 and an int32's count), so index arithmetic has 32 bits.
struct PageMap {
  const int32_t* block_table;
  uint32_t page_size, num_pages, max_pages;
  // Entry `pidx` of sequence row b, or -1 past the row.
  __device__ __forceinline__ int entry(int b, uint32_t pidx) const {
    return pidx >= max_pages ? -1 : block_table[(size_t)b * max_pages + pidx];
  }
};

struct Int4AppendArgs {
  const __half* new_k;  // [B, T, Hkv, 128]
  const __half* new_v;
  uint8_t* k_pool;  // blocks [num_pages, Hkv, page_size / 16]
  uint8_t* v_pool;
  const int32_t* positions;
  int32_t* status;
  const float* freq_cis;
  PageMap map;
  int n_tokens, num_kv_heads, rope_positions;
};

// Of a CTA: warps share nothing, and at the append's 90 registers CTAs of 4 leave 20
// of them resident on an SM where CTAs of 8 leave 16 (32 x 512 tokens written and
// read: 35.5 us against 39.1; 2 warps 35.4, but 7.6 against 7.1 for 32 x 1 tokens).
constexpr int kWarps = 4;

// One warp per (sequence, 16-token block, kv head, K or V).  Half-warp hw takes the
// token pairs 2 j + hw, lane l16 the dims [8 l16, 8 l16 + 8): one K word per token
// and two V words per pair; a group's maximum is four lanes'.  All 16 rows (4 KB)
// are loaded before any is quantised.  (A lane for a whole group of two tokens saves a
// seventh of the instructions, 32.3 us against 33.7 for 32 x 512 tokens, but has four
// times the RoPE work in a row: 11.1 against 10.0 for 1 x 8191, 7.3 against 6.5 for 32 x 1.)
struct BlockWork {
  int b, h, kv;
  long long first;   // the block's first position
  int lo, hi;        // its tokens in the chunk: [lo, hi) of 16
  long long row0;    // row of token 0 in [B, T, Hkv] (of lo > 0: before the chunk's)
  int entry, tile;   // of the block table, not yet looked at; the block within its page
  __device__ __forceinline__ bool whole() const { return lo == 0 && hi == 16; }
};
// False: nothing of the chunk is there.
__device__ __forceinline__ bool find_block(BlockWork& w, const PageMap& map, const int32_t* positions, int n_tokens,
                                           int heads, int wid) {
  const int pair = wid >> 1, nth = pair / heads;
  w.kv = wid & 1;
  w.h = pair - nth * heads;
  w.b = blockIdx.y;
  const int pos0 = positions[w.b];
  w.first = (long long)(pos0 & ~15) + 16ll * nth;
  const long long end = (long long)pos0 + n_tokens;
  if (w.first >= end) return false;
  w.lo = (int)max(0ll, pos0 - w.first);
  w.hi = (int)min(16ll, end - w.first);
  w.row0 = ((long long)w.b * n_tokens + (w.first - pos0)) * heads + w.h;
  const uint32_t tile = (uint32_t)w.first / 16, per = map.page_size / 16, pidx = tile / per;
  w.entry = pos0 < 0 ? -1 : map.entry(w.b, pidx);
  w.tile = (int)(tile - pidx * per);
  return true;
}
// The block's byte offset in the pool.  False, and reported: it is not mapped.
__device__ __forceinline__ bool mapped(const BlockWork& w, const PageMap& map, int heads, int32_t* status,
                                       size_t& block) {
  block = (((size_t)(unsigned)w.entry * heads + w.h) * (map.page_size / 16) + w.tile) * kI4Block;
  if ((uint32_t)w.entry < map.num_pages) return true;
  if ((threadIdx.x & 31) == 0) report(status, DOE_DEVICE_ERR_PAGE);
  return false;
}

// WHOLE: all 16 tokens are in the chunk.
template <bool ROPE, bool WHOLE>
__device__ __forceinline__ void append_block(const Int4AppendArgs& a, const BlockWork& w) {
  const int lane = threadIdx.x & 31, hw = lane >> 4, l16 = lane & 15, t = l16 & 3, group = l16 >> 2;
  const __half* src = (w.kv ? a.new_v : a.new_k) + w.row0 * 128 + 8 * l16;
  const int stride = a.num_kv_heads * 128;  // of a token
  auto live = [&](int tok) { return WHOLE || (tok >= w.lo && tok < w.hi); };
  uint4 x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int tok = 4 * (i >> 1) + 2 * hw + (i & 1);
    x[i] = make_uint4(0, 0, 0, 0);
    if (live(tok)) x[i] = __ldcs(reinterpret_cast<const uint4*>(src + (long long)tok * stride));
  }
  size_t block;  // the rows are on their way while the page is looked up
  if (!mapped(w, a.map, a.num_kv_heads, a.status, block)) return;
  uint8_t* dst = (w.kv ? a.v_pool : a.k_pool) + block;
  if (ROPE && w.kv == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int tok = 4 * (i >> 1) + 2 * hw + (i & 1);
      uint4 p;
      p.x = __shfl_xor_sync(0xffffffffu, x[i].x, 8);
      p.y = __shfl_xor_sync(0xffffffffu, x[i].y, 8);
      p.z = __shfl_xor_sync(0xffffffffu, x[i].z, 8);
      p.w = __shfl_xor_sync(0xffffffffu, x[i].w, 8);
      if (live(tok)) {
        float c[8], sn[8];
        rope_table<4>(a.freq_cis, a.rope_positions, 64, w.first + tok, 8 * (l16 & 7), a.status, l16 == 0, c, sn);
        const uint4 mine = x[i];
        rope_rotate<4>(reinterpret_cast<const uint32_t*>(&mine), reinterpret_cast<const uint32_t*>(&p), l16 < 8, c, sn,
                       reinterpret_cast<uint32_t*>(&x[i]));
      }
    }
  }
  // scales of all rows first; the codes' two forms (see quantize_u4x2) then differ
  // once per warp.  A NaN makes its group's scale NaN, so the group reads back as NaN
  float s[8], rs[8];
  __half sh[8];
  bool normal = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2* hx = reinterpret_cast<const __half2*>(&x[i]);
    __half2 m2 = __hmax2_nan(__hmax2_nan(__habs2(hx[0]), __habs2(hx[1])), __hmax2_nan(__habs2(hx[2]), __habs2(hx[3])));
    uint32_t m = *reinterpret_cast<uint32_t*>(&m2), o = __shfl_xor_sync(0xffffffffu, m, 1);
    m2 = __hmax2_nan(m2, *reinterpret_cast<__half2*>(&o));
    m = *reinterpret_cast<uint32_t*>(&m2);
    o = __shfl_xor_sync(0xffffffffu, m, 2);
    m2 = __hmax2_nan(m2, *reinterpret_cast<__half2*>(&o));
    sh[i] = __float2half_rn(div7(__half2float(__hmax_nan(__low2half(m2), __high2half(m2)))));
    s[i] = __half2float(sh[i]);
    rs[i] = inverse_of(s[i]);
    normal &= s[i] >= 0x1p-14f;
  }
  normal = __all_sync(0xffffffffu, normal);
  auto codes = [&](auto clamp, int i, uint2 (&c)[4]) {
    const __half2* hx = reinterpret_cast<const __half2*>(&x[i]);
#pragma unroll
    for (int d = 0; d < 4; ++d) c[d] = quantize_u4x2<decltype(clamp)::value>(__half22float2(hx[d]), s[i], rs[i]);
  };
  auto write = [&](auto clamp) {
    if (w.kv == 0) {
      uint8_t* at = dst + hw * 128 + t * 16 + group * 4;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int tok = 4 * (i >> 1) + (i & 1);  // + 2 hw
        uint2 c[4];
        codes(clamp, i, c);
        const uint32_t even = pack_u4x4(c[0].x, c[1].x, c[2].x, c[3].x);
        const uint32_t odd = pack_u4x4(c[0].y, c[1].y, c[2].y, c[3].y);
        if (live(tok + 2 * hw)) {
          *reinterpret_cast<uint32_t*>(at + tok * 64) = prmt(even, odd, 0x5410u);
          if (t == 0) reinterpret_cast<__half*>(dst + kI4Codes)[(tok + 2 * hw) * 4 + group] = sh[i];
        }
      }
      return;
    }
    // dims 8 l16 .. + 8 are g = 2 t (the first four) and g = 2 t + 1
    uint8_t* at = dst + t * 128 + hw * 16 + group * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // pair 2 j + hw
      uint2 c[2][4];
      codes(clamp, 2 * j, c[0]);
      codes(clamp, 2 * j + 1, c[1]);
      const bool live0 = live(4 * j + 2 * hw), live1 = live(4 * j + 2 * hw + 1);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t half[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          half[e] = pack_u4x4(c[e][2 * u].x, c[e][2 * u].y, c[e][2 * u + 1].x, c[e][2 * u + 1].y);
        uint8_t* to = at + (j >> 1) * 512 + (j & 1) * 32 + u * 64;
        if (WHOLE || (live0 && live1)) {
          *reinterpret_cast<uint32_t*>(to) = prmt(half[0], half[1], 0x5410u);
        } else {
          if (live0) *reinterpret_cast<uint16_t*>(to) = (uint16_t)half[0];
          if (live1) *reinterpret_cast<uint16_t*>(to + 2) = (uint16_t)half[1];
        }
      }
      if (t == 0) {
        __half* to = reinterpret_cast<__half*>(dst + kI4Codes) + ((2 * j + hw) * 4 + group) * 2;
        if (WHOLE) {
          *reinterpret_cast<__half2*>(to) = __halves2half2(sh[2 * j], sh[2 * j + 1]);
        } else {
          if (live0) to[0] = sh[2 * j];
          if (live1) to[1] = sh[2 * j + 1];
        }
      }
    }
  };
  if (normal) write(std::false_type());
  else write(std::true_type());
}

template <bool ROPE>
__global__ void __launch_bounds__(kWarps * 32) int4_append_kernel(const Int4AppendArgs a, int warps_per_seq) {
  pdl_wait();
  pdl_trigger();
  const int wid = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (wid >= warps_per_seq) return;
  BlockWork w;
  if (!find_block(w, a.map, a.positions, a.n_tokens, a.num_kv_heads, wid)) return;
  if (w.whole()) append_block<ROPE, true>(a, w);
  else append_block<ROPE, false>(a, w);
}

int launch_int4_append(const doe_paged_kv* kv, uint32_t num_seqs, uint32_t n_tokens, const void* new_k,
                       const void* new_v, const int32_t* positions, const float* freq_cis, uint32_t rope_positions,
                       const doe_launch* launch) {
  if (num_seqs == 0 || n_tokens == 0) return DOE_OK;
  Int4AppendArgs a;
  a.new_k = static_cast<const __half*>(new_k);
  a.new_v = static_cast<const __half*>(new_v);
  a.k_pool = static_cast<uint8_t*>(kv->k_pool);
  a.v_pool = static_cast<uint8_t*>(kv->v_pool);
  a.positions = positions;
  a.status = launch->status;
  a.freq_cis = freq_cis;
  a.map = {kv->block_table, kv->page_size, kv->num_pages, kv->max_pages_per_seq};
  a.n_tokens = (int)n_tokens;
  a.num_kv_heads = (int)kv->num_kv_heads;
  a.rope_positions = (int)rope_positions;
  // a chunk starting inside a block touches one block more
  const uint64_t warps = (((uint64_t)n_tokens + 14) / 16 + 1) * kv->num_kv_heads * 2;
  const dim3 grid((unsigned)((warps + kWarps - 1) / kWarps), num_seqs);
  cudaStream_t st = static_cast<cudaStream_t>(launch->stream);
  return cuda_status(launch_pdl(freq_cis != nullptr ? int4_append_kernel<true> : int4_append_kernel<false>, grid,
                                dim3(kWarps * 32), 0, st, a, (int)warps),
                     "int4_append_kernel");
}

// ---- read: rows [positions[b], + T) of every sequence as values ---------------
struct PagedReadArgs {
  const uint8_t* pool[2];
  const __half* scale[2];  // int8: [num_pages, Hkv, page_size]
  void* out[2];            // [B, T, Hkv, D]
  const int32_t* positions;
  int32_t* status;
  PageMap map;
  int n_tokens, num_kv_heads, head_dim;
};

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight consecutive values, rounded to T, in 16-byte stores.
template <typename T>
__device__ __forceinline__ void store8(T* dst, const float (&v)[8]) {
  alignas(16) T r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = from_f32<T>(v[i]);
#pragma unroll
  for (int i = 0; i < (int)sizeof(r) / 16; ++i)
    reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(r)[i];
}

// (n - 8) * s of a code pair where the mask has left it, in f16: 1024 + n (or 1024 +
// 16 n) and n - 8 are exact, so the product is rounded once, as from f32.
__device__ __forceinline__ __half2 code_values(uint32_t w, int i, __half2 s) {
  const uint32_t x = (i & 2) ? w >> 8 : w;
  uint32_t m = (i & 1) ? (x & 0x00f000f0u) | 0x64006400u : (x & 0x000f000fu) | 0x64006400u;
  __half2 v = *reinterpret_cast<__half2*>(&m);
  v = (i & 1) ? __hfma2(v, __float2half2_rn(0.0625f), __float2half2_rn(-72.0f)) : __hadd2(v, __float2half2_rn(-1032.0f));
  return __hmul2(v, s);
}

// The lane layout of append_block, reversed.
template <typename T, bool WHOLE>
__device__ __forceinline__ void read_block(const PagedReadArgs& a, const BlockWork& w) {
  const int lane = threadIdx.x & 31, hw = lane >> 4, l16 = lane & 15, t = l16 & 3, group = l16 >> 2;
  size_t block;
  const bool some = mapped(w, a.map, a.num_kv_heads, a.status, block);
  const uint8_t* src = (w.kv ? a.pool[1] : a.pool[0]) + (some ? block : 0);
  T* dst = static_cast<T*>(w.kv ? a.out[1] : a.out[0]) + w.row0 * 128 + 8 * l16;
  const int stride = a.num_kv_heads * 128;  // of a token
  auto live = [&](int tok) { return WHOLE || (tok >= w.lo && tok < w.hi); };
  // words and scales of tokens 4 j + 2 hw and the next (V: of their pair)
  uint32_t code[4][2];
  __half2 s[4];
  const uint8_t* at = src + group * 4 + (w.kv ? t * 128 + hw * 16 : hw * 128 + t * 16);
  const __half* sc = reinterpret_cast<const __half*>(src + kI4Codes) + (w.kv ? hw * 8 + group * 2 : hw * 8 + group);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (!some) {  // reads as zeros
      code[j][0] = code[j][1] = 0u;
      s[j] = __float2half2_rn(0.0f);
    } else if (w.kv) {
      const uint8_t* v = at + (j >> 1) * 512 + (j & 1) * 32;
      code[j][0] = *reinterpret_cast<const uint32_t*>(v);
      code[j][1] = *reinterpret_cast<const uint32_t*>(v + 64);
      s[j] = *reinterpret_cast<const __half2*>(sc + j * 16);
    } else {
      code[j][0] = *reinterpret_cast<const uint32_t*>(at + j * 256);
      code[j][1] = *reinterpret_cast<const uint32_t*>(at + j * 256 + 64);
      s[j] = __halves2half2(sc[j * 16], sc[j * 16 + 4]);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int tok = 4 * j + 2 * hw;
    T* to = dst + (long long)tok * stride;
    if constexpr (std::is_same<T, __half>::value) {
      // both tokens' values as four (dim, dim + 1) pairs
      __half2 v[2][4];
      if (w.kv == 0) {
        const __half2 s0 = __low2half2(s[j]), s1 = __high2half2(s[j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[0][i] = code_values(code[j][0], i, s0);
          v[1][i] = code_values(code[j][1], i, s1);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; i += 2)
#pragma unroll
          for (int u = 0; u < 2; ++u) {  // one dim of both tokens each
            const __half2 a0 = code_values(code[j][u], i, s[j]), a1 = code_values(code[j][u], i + 1, s[j]);
            v[0][2 * u + i / 2] = __lows2half2(a0, a1);
            v[1][2 * u + i / 2] = __highs2half2(a0, a1);
          }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (live(tok + e)) __stcs(reinterpret_cast<uint4*>(to + e * stride), *reinterpret_cast<const uint4*>(v[e]));
    } else {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (!live(tok + e)) continue;
        const float sf = e ? __high2float(s[j]) : __low2float(s[j]);
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t n = w.kv == 0 ? (code[j][e] >> (4 * (i >> 1) + 16 * (i & 1))) & 15u
                                       : (code[j][i >> 2] >> (16 * e + 4 * (i & 3))) & 15u;
          f[i] = (float)((int)n - 8) * sf;
        }
        store8(to + e * stride, f);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) int4_read_kernel(const PagedReadArgs a, int warps_per_seq) {
  pdl_wait();
  pdl_trigger();
  const int wid = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (wid >= warps_per_seq) return;
  BlockWork w;
  if (!find_block(w, a.map, a.positions, a.n_tokens, a.num_kv_heads, wid)) return;
  if (w.whole()) read_block<T, true>(a, w);
  else read_block<T, false>(a, w);
}

// f16 and int8 rows: one warp per (sequence, token), lanes over Hkv * D in
// runs of 8.  Bound by HBM writes and, for int8, by a scale load per run: 32 x 512 tokens
// of 8 kv heads as f16 take 26.8 us from f16 pools (134 MB, 0.77 of the measured copy
// rate), 25.8 from int8 (101 MB, 0.60).
template <typename T, bool INT8>
__global__ void __launch_bounds__(256) paged_read_kernel(const PagedReadArgs a) {
  const int tok = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, b = blockIdx.y;
  if (tok >= a.n_tokens) return;
  const int pos0 = a.positions[b];
  const uint32_t pos = (uint32_t)pos0 + tok, pidx = pos / a.map.page_size;
  int page = pos0 < 0 ? -1 : a.map.entry(b, pidx);
  if ((uint32_t)page >= a.map.num_pages) {
    page = -1;
    if (lane == 0) report(a.status, DOE_DEVICE_ERR_PAGE);
  }
  const int in_page = (int)(pos - pidx * a.map.page_size);
  const int Hkv = a.num_kv_heads, D = a.head_dim, n = Hkv * D;
  const size_t row = ((size_t)page * a.map.page_size + in_page) * n;
  const size_t out = ((size_t)b * a.n_tokens + tok) * n;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    T* dst = static_cast<T*>(a.out[kv]) + out;
    for (int i = lane * 8; i < n; i += 256) {
      float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};  // of an unmapped page
      if (page < 0) {
      } else if (INT8) {
        const float s = __half2float(a.scale[kv][((size_t)page * Hkv + i / D) * a.map.page_size + in_page]);
        const uint2 w = *reinterpret_cast<const uint2*>(a.pool[kv] + row + i);
        const int8_t* c = reinterpret_cast<const int8_t*>(&w);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (float)c[k] * s;
      } else {
        const uint4 w = *reinterpret_cast<const uint4*>(a.pool[kv] + (row + i) * 2);
        const __half2* c = reinterpret_cast<const __half2*>(&w);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = __half22float2(c[k]);
          v[2 * k] = f.x;
          v[2 * k + 1] = f.y;
        }
      }
      store8(dst + i, v);
    }
  }
}

template <typename T>
static int launch_read(const doe_paged_kv* kv, const PagedReadArgs& a, uint32_t num_seqs, cudaStream_t st) {
  if (kv->kv_dtype == DOE_KV_INT4) {
    const uint64_t warps = (((uint64_t)a.n_tokens + 14) / 16 + 1) * kv->num_kv_heads * 2;
    const dim3 grid((unsigned)((warps + kWarps - 1) / kWarps), num_seqs);
    return cuda_status(launch_pdl(int4_read_kernel<T>, grid, dim3(kWarps * 32), 0, st, a, (int)warps),
                       "int4_read_kernel");
  }
  const dim3 grid(((uint32_t)a.n_tokens + 7) / 8, num_seqs);
  if (kv->kv_dtype == DOE_KV_INT8)
    paged_read_kernel<T, true><<<grid, 256, 0, st>>>(a);
  else
    paged_read_kernel<T, false><<<grid, 256, 0, st>>>(a);
  return cuda_status(cudaGetLastError(), "paged_read_kernel");
}

int launch_paged_read(const doe_paged_kv* kv, uint32_t num_seqs, uint32_t n_tokens, const int32_t* positions,
                      void* k_out, void* v_out, uint32_t dtype, const doe_launch* launch) {
  if (num_seqs == 0 || n_tokens == 0) return DOE_OK;
  PagedReadArgs a;
  a.pool[0] = static_cast<const uint8_t*>(kv->k_pool);
  a.pool[1] = static_cast<const uint8_t*>(kv->v_pool);
  a.scale[0] = static_cast<const __half*>(kv->k_scale);
  a.scale[1] = static_cast<const __half*>(kv->v_scale);
  a.out[0] = k_out;
  a.out[1] = v_out;
  a.positions = positions;
  a.status = launch->status;
  a.map = {kv->block_table, kv->page_size, kv->num_pages, kv->max_pages_per_seq};
  a.n_tokens = (int)n_tokens;
  a.num_kv_heads = (int)kv->num_kv_heads;
  a.head_dim = (int)kv->head_dim;
  cudaStream_t st = static_cast<cudaStream_t>(launch->stream);
  switch (dtype) {
    case DOE_DTYPE_F32: return launch_read<float>(kv, a, num_seqs, st);
    case DOE_DTYPE_BF16: return launch_read<__nv_bfloat16>(kv, a, num_seqs, st);
    default: return launch_read<__half>(kv, a, num_seqs, st);
  }
}

}  // namespace doe
