// kv_int4.cu -- writes into and reads out of the 4-bit paged KV cache.
//
//   append : f16 rows [B, T, Hkv, 128], K optionally rotated (rope.wgsl:12-35),
//            quantised into the blocks of int4.cuh
//   read   : value rows of any cache type (f16, int8, int4) as f16, bf16 or f32
//
// Both are copies with a little arithmetic, bound by HBM: 512 bytes of f16 K
// and V against 144 bytes of blocks per (token, kv head).
#include <type_traits>

#include "int4.cuh"

namespace doe {

// Page of token `pos` of sequence row b, or -1.
struct PageMap {
  const int32_t* block_table;
  int page_size, num_pages, max_pages;
  __device__ __forceinline__ int page(int b, long long pos) const {
    const long long pidx = pos / page_size;
    if (pos < 0 || pidx >= max_pages) return -1;
    const int p = block_table[(size_t)b * max_pages + pidx];
    return (unsigned)p < (unsigned)num_pages ? p : -1;
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

// One warp per (sequence, 16-token block, kv head, K or V).  Half-warp hw takes the
// token pairs 2 j + hw, lane l16 the dims [8 l16, 8 l16 + 8): one K word per token
// and two V words per pair; a group's maximum is four lanes'.  All 16 rows (4 KB)
// are loaded before any is quantised.
struct BlockWork {
  int b, h, kv;
  int pos0;             // the chunk's first position
  long long first, end;  // the block's first position, the chunk's end
  size_t block;         // byte offset in the pool
  bool mapped;
  __device__ __forceinline__ bool live(int tok) const { return first + tok >= pos0 && first + tok < end; }
  __device__ __forceinline__ size_t row(int tok, int n_tokens, int heads) const {
    return ((size_t)b * n_tokens + (size_t)(first + tok - pos0)) * heads + h;
  }
};
// False: nothing of the chunk is there.  An unmapped block is reported.
__device__ __forceinline__ bool find_block(BlockWork& w, const PageMap& map, const int32_t* positions, int n_tokens,
                                           int heads, int wid, int32_t* status) {
  w.kv = wid & 1;
  w.h = (wid >> 1) % heads;
  w.b = blockIdx.y;
  w.pos0 = positions[w.b];
  w.first = (long long)(w.pos0 & ~15) + 16ll * (wid / (2 * heads));
  w.end = (long long)w.pos0 + n_tokens;
  if (w.first >= w.end) return false;
  const int page = w.pos0 < 0 ? -1 : map.page(w.b, w.first);
  w.mapped = page >= 0;
  if (!w.mapped && (threadIdx.x & 31) == 0) report(status, DOE_DEVICE_ERR_PAGE);
  const int tile = (int)(w.first % map.page_size) / 16;
  w.block = w.mapped ? (((size_t)page * heads + w.h) * (map.page_size / 16) + tile) * kI4Block : 0;
  return true;
}

template <bool ROPE>
__global__ void __launch_bounds__(256) int4_append_kernel(const Int4AppendArgs a, int warps_per_seq) {
  const int wid = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (wid >= warps_per_seq) return;
  const int hw = lane >> 4, l16 = lane & 15, t = l16 & 3, group = l16 >> 2;
  BlockWork w;
  if (!find_block(w, a.map, a.positions, a.n_tokens, a.num_kv_heads, wid, a.status) || !w.mapped) return;
  const __half* src = (w.kv ? a.new_v : a.new_k) + 8 * l16;
  uint8_t* dst = (w.kv ? a.v_pool : a.k_pool) + w.block;
  uint4 x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int tok = 4 * (i >> 1) + 2 * hw + (i & 1);
    x[i] = make_uint4(0, 0, 0, 0);
    if (w.live(tok)) x[i] = __ldcs(reinterpret_cast<const uint4*>(src + w.row(tok, a.n_tokens, a.num_kv_heads) * 128));
  }
  if (ROPE && w.kv == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int tok = 4 * (i >> 1) + 2 * hw + (i & 1);
      uint4 p;
      p.x = __shfl_xor_sync(0xffffffffu, x[i].x, 8);
      p.y = __shfl_xor_sync(0xffffffffu, x[i].y, 8);
      p.z = __shfl_xor_sync(0xffffffffu, x[i].z, 8);
      p.w = __shfl_xor_sync(0xffffffffu, x[i].w, 8);
      if (w.live(tok)) {
        float c[8], sn[8];
        rope_table<4>(a.freq_cis, a.rope_positions, 64, w.first + tok, 8 * (l16 & 7), a.status, l16 == 0, c, sn);
        const uint4 mine = x[i];
        rope_rotate<4>(reinterpret_cast<const uint32_t*>(&mine), reinterpret_cast<const uint32_t*>(&p), l16 < 8, c, sn,
                       reinterpret_cast<uint32_t*>(&x[i]));
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int pair = 2 * j + hw;
    uint2 c[2][4];  // codes of dims (2 i, 2 i + 1)
    __half sh[2];
    bool live[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      live[e] = w.live(2 * pair + e);
      const __half2* hx = reinterpret_cast<const __half2*>(&x[2 * j + e]);
      const __half2 m2 = __hmax2(__hmax2(__habs2(hx[0]), __habs2(hx[1])), __hmax2(__habs2(hx[2]), __habs2(hx[3])));
      float amax = fmaxf(__low2float(m2), __high2float(m2));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      sh[e] = __float2half_rn(div7(amax));
      const float s = __half2float(sh[e]), rs = inverse_of(s);
      if (s >= 0x1p-14f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c[e][i] = quantize_u4x2<false>(__half22float2(hx[i]), s, rs);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) c[e][i] = quantize_u4x2<true>(__half22float2(hx[i]), s, rs);
      }
    }
    if (w.kv == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int tok = 2 * pair + e;
        const uint32_t even = pack_u4x4(c[e][0].x, c[e][1].x, c[e][2].x, c[e][3].x);
        const uint32_t odd = pack_u4x4(c[e][0].y, c[e][1].y, c[e][2].y, c[e][3].y);
        if (live[e]) {
          *reinterpret_cast<uint32_t*>(dst + tok * 64 + t * 16 + group * 4) = prmt(even, odd, 0x5410u);
          if (t == 0) *reinterpret_cast<__half*>(dst + kI4Codes + (tok * 4 + group) * 2) = sh[e];
        }
      }
    } else {
      // dims 8 l16 .. + 8 are g = 2 t (the first four) and g = 2 t + 1
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t half[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          half[e] = pack_u4x4(c[e][2 * u].x, c[e][2 * u].y, c[e][2 * u + 1].x, c[e][2 * u + 1].y);
        uint8_t* at = dst + (((pair >> 2) * 8 + 2 * t + u) * 4 + (pair & 3)) * 16 + group * 4;
        if (live[0] && live[1]) {
          *reinterpret_cast<uint32_t*>(at) = prmt(half[0], half[1], 0x5410u);
        } else {
          if (live[0]) *reinterpret_cast<uint16_t*>(at) = (uint16_t)half[0];
          if (live[1]) *reinterpret_cast<uint16_t*>(at + 2) = (uint16_t)half[1];
        }
      }
      if (t == 0) {
        __half* at = reinterpret_cast<__half*>(dst + kI4Codes) + (pair * 4 + group) * 2;
        if (live[0]) at[0] = sh[0];
        if (live[1]) at[1] = sh[1];
      }
    }
  }
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
  a.map = {kv->block_table, (int)kv->page_size, (int)kv->num_pages, (int)kv->max_pages_per_seq};
  a.n_tokens = (int)n_tokens;
  a.num_kv_heads = (int)kv->num_kv_heads;
  a.rope_positions = (int)rope_positions;
  // a chunk starting inside a block touches one block more
  const uint64_t warps = (((uint64_t)n_tokens + 14) / 16 + 1) * kv->num_kv_heads * 2;
  const dim3 grid((unsigned)((warps + 7) / 8), num_seqs);
  cudaStream_t st = static_cast<cudaStream_t>(launch->stream);
  if (freq_cis != nullptr)
    int4_append_kernel<true><<<grid, 256, 0, st>>>(a, (int)warps);
  else
    int4_append_kernel<false><<<grid, 256, 0, st>>>(a, (int)warps);
  return cuda_status(cudaGetLastError(), "int4_append_kernel");
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

// The lane layout of int4_append_kernel, reversed.
template <typename T>
__global__ void __launch_bounds__(256) int4_read_kernel(const PagedReadArgs a, int warps_per_seq) {
  const int wid = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (wid >= warps_per_seq) return;
  const int hw = lane >> 4, l16 = lane & 15, t = l16 & 3, group = l16 >> 2;
  BlockWork w;
  if (!find_block(w, a.map, a.positions, a.n_tokens, a.num_kv_heads, wid, a.status)) return;
  const uint8_t* src = (w.kv ? a.pool[1] : a.pool[0]) + w.block;
  T* dst = static_cast<T*>(w.kv ? a.out[1] : a.out[0]) + 8 * l16;
  uint32_t code[4][2];
  __half s[4][2];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int pair = 2 * j + hw;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int tok = 2 * pair + e;
      const int at = w.kv ? (((pair >> 2) * 8 + 2 * t + e) * 4 + (pair & 3)) * 16 + group * 4 : tok * 64 + t * 16 + group * 4;
      const int sc = w.kv ? (pair * 4 + group) * 2 + e : tok * 4 + group;
      // an unmapped block reads as zeros
      code[j][e] = w.mapped ? *reinterpret_cast<const uint32_t*>(src + at) : 0u;
      s[j][e] = w.mapped ? reinterpret_cast<const __half*>(src + kI4Codes)[sc] : __ushort_as_half(0);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // values of tokens 2 pair and 2 pair + 1 as four (dim, dim + 1) pairs
    __half2 v[2][4];
    if constexpr (sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value) {
      if (w.kv == 0) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[e][i] = code_values(code[j][e], i, __half2half2(s[j][e]));
      } else {
        const __half2 s2 = __halves2half2(s[j][0], s[j][1]);
#pragma unroll
        for (int i = 0; i < 4; i += 2)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            // one dim of both tokens each
            const __half2 a0 = code_values(code[j][u], i, s2), a1 = code_values(code[j][u], i + 1, s2);
            v[0][2 * u + i / 2] = __lows2half2(a0, a1);
            v[1][2 * u + i / 2] = __highs2half2(a0, a1);
          }
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int tok = 2 * (2 * j + hw) + e;
      if (!w.live(tok)) continue;
      T* at = dst + w.row(tok, a.n_tokens, a.num_kv_heads) * 128;
      if constexpr (sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value) {
        __stcs(reinterpret_cast<uint4*>(at), *reinterpret_cast<const uint4*>(v[e]));
      } else {
        const float sf = __half2float(s[j][e]);
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t n = w.kv == 0 ? (code[j][e] >> (4 * (i >> 1) + 16 * (i & 1))) & 15u
                                       : (code[j][i >> 2] >> (16 * e + 4 * (i & 3))) & 15u;
          f[i] = (float)((int)n - 8) * sf;
        }
        store8(at, f);
      }
    }
  }
}

// f16 and int8 rows: one warp per (sequence, token), lanes over Hkv * D in
// runs of 8.
template <typename T, bool INT8>
__global__ void __launch_bounds__(256) paged_read_kernel(const PagedReadArgs a) {
  const int tok = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, b = blockIdx.y;
  if (tok >= a.n_tokens) return;
  const int pos0 = a.positions[b];
  const long long pos = (long long)pos0 + tok;
  const int page = pos0 < 0 ? -1 : a.map.page(b, pos);
  if (page < 0 && lane == 0) report(a.status, DOE_DEVICE_ERR_PAGE);
  const int in_page = (int)(pos % a.map.page_size);
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
    const dim3 grid((unsigned)((warps + 7) / 8), num_seqs);
    int4_read_kernel<T><<<grid, 256, 0, st>>>(a, (int)warps);
    return cuda_status(cudaGetLastError(), "int4_read_kernel");
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
  a.map = {kv->block_table, (int)kv->page_size, (int)kv->num_pages, (int)kv->max_pages_per_seq};
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
