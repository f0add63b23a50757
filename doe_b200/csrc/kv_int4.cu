// kv_int4.cu -- writes into and reads out of the 4-bit paged KV cache.
//
//   append : f16 rows [B, T, Hkv, 128], K optionally rotated (rope.wgsl:12-35),
//            quantised into the blocks of int4.cuh
//   read   : value rows of any cache type (f16, int8, int4) as f16, bf16 or f32
//
// Both are copies with a little arithmetic, bound by HBM: 512 bytes of f16 K
// and V against 144 bytes of blocks per (token, kv head).
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

// One warp per (sequence, 16-token block, kv head); half-warp hw takes the
// token pairs 2 j + hw, lane l16 the dims [8 l16, 8 l16 + 8): one K word per
// token and two V words per pair.
__global__ void __launch_bounds__(256) int4_append_kernel(const Int4AppendArgs a, int warps_per_seq) {
  const int wid = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (wid >= warps_per_seq) return;
  const int hw = lane >> 4, l16 = lane & 15, t = l16 & 3, group = l16 >> 2;
  const int Hkv = a.num_kv_heads, h = wid % Hkv, b = blockIdx.y;
  const int pos0 = a.positions[b];
  if (pos0 < 0) {
    if (wid == 0 && lane == 0) report(a.status, DOE_DEVICE_ERR_PAGE);
    return;
  }
  const long long first = (long long)(pos0 & ~15) + 16ll * (wid / Hkv);  // the block's first position
  const long long end = (long long)pos0 + a.n_tokens;
  if (first >= end) return;
  const int page = a.map.page(b, first);
  if (page < 0) {
    if (lane == 0) report(a.status, DOE_DEVICE_ERR_PAGE);
    return;
  }
  const int tiles = a.map.page_size / 16;
  const int tile = (int)(first % a.map.page_size) / 16;
  const size_t block = (((size_t)page * Hkv + h) * tiles + tile) * kI4Block;

  for (int kv = 0; kv < 2; ++kv) {
    const __half* src = kv ? a.new_v : a.new_k;
    uint8_t* dst = (kv ? a.v_pool : a.k_pool) + block;
    uint4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // token 2 (2 (i / 2) + hw) + i % 2 of the block
      const int tok = 4 * (i >> 1) + 2 * hw + (i & 1);
      const long long pos = first + tok;
      const bool live = pos >= pos0 && pos < end;
      x[i] = make_uint4(0, 0, 0, 0);
      if (live)
        x[i] = *reinterpret_cast<const uint4*>(
            src + (((size_t)b * a.n_tokens + (size_t)(pos - pos0)) * Hkv + h) * 128 + 8 * l16);
    }
    if (kv == 0 && a.freq_cis != nullptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int tok = 4 * (i >> 1) + 2 * hw + (i & 1);
        const long long pos = first + tok;
        const bool live = pos >= pos0 && pos < end;
        uint4 p;
        p.x = __shfl_xor_sync(0xffffffffu, x[i].x, 8);
        p.y = __shfl_xor_sync(0xffffffffu, x[i].y, 8);
        p.z = __shfl_xor_sync(0xffffffffu, x[i].z, 8);
        p.w = __shfl_xor_sync(0xffffffffu, x[i].w, 8);
        if (live) {
          float c[8], sn[8];
          rope_table<4>(a.freq_cis, a.rope_positions, 64, pos, 8 * (l16 & 7), a.status, l16 == 0, c, sn);
          const uint4 mine = x[i];
          rope_rotate<4>(reinterpret_cast<const uint32_t*>(&mine), reinterpret_cast<const uint32_t*>(&p), l16 < 8, c,
                         sn, reinterpret_cast<uint32_t*>(&x[i]));
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int pair = 2 * j + hw;
      uint32_t code[2][8];
      __half sh[2];
      bool live[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const long long pos = first + 2 * pair + e;
        live[e] = pos >= pos0 && pos < end;
        const __half2* hx = reinterpret_cast<const __half2*>(&x[2 * j + e]);
        __half2 m2 = __hmax2(__hmax2(__habs2(hx[0]), __habs2(hx[1])), __hmax2(__habs2(hx[2]), __habs2(hx[3])));
        float amax = fmaxf(__low2float(m2), __high2float(m2));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        sh[e] = __float2half_rn(div7(amax));
        const float s = __half2float(sh[e]);
        const float rs = s != 0.0f ? __frcp_rn(s) : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = __half22float2(hx[i]);
          code[e][2 * i] = s != 0.0f ? quantize_u4(f.x, s, rs) : 8u;
          code[e][2 * i + 1] = s != 0.0f ? quantize_u4(f.y, s, rs) : 8u;
        }
      }
      if (kv == 0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t w = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) w |= (code[e][2 * i] | (code[e][2 * i + 1] << 16)) << (4 * i);
          const int tok = 2 * pair + e;
          if (live[e]) {
            *reinterpret_cast<uint32_t*>(dst + tok * 64 + t * 16 + group * 4) = w;
            if (t == 0) *reinterpret_cast<__half*>(dst + kI4Codes + (tok * 4 + group) * 2) = sh[e];
          }
        }
      } else {
        // dims 8 l16 .. + 8 are g = 2 t (the first four) and g = 2 t + 1
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t hw16[2];
#pragma unroll
          for (int e = 0; e < 2; ++e)
            hw16[e] = code[e][4 * u] | (code[e][4 * u + 1] << 4) | (code[e][4 * u + 2] << 8) | (code[e][4 * u + 3] << 12);
          uint8_t* at = dst + (((pair >> 2) * 8 + 2 * t + u) * 4 + (pair & 3)) * 16 + group * 4;
          if (live[0] && live[1]) {
            *reinterpret_cast<uint32_t*>(at) = hw16[0] | (hw16[1] << 16);
          } else {
            if (live[0]) *reinterpret_cast<uint16_t*>(at) = (uint16_t)hw16[0];
            if (live[1]) *reinterpret_cast<uint16_t*>(at + 2) = (uint16_t)hw16[1];
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
  const uint64_t warps = (((uint64_t)n_tokens + 14) / 16 + 1) * kv->num_kv_heads;
  const dim3 grid((unsigned)((warps + 7) / 8), num_seqs);
  int4_append_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(launch->stream)>>>(a, (int)warps);
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

// The lane layout of int4_append_kernel, reversed: one warp per (sequence,
// 16-token block, kv head).
template <typename T>
__global__ void __launch_bounds__(256) int4_read_kernel(const PagedReadArgs a, int warps_per_seq) {
  const int wid = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (wid >= warps_per_seq) return;
  const int hw = lane >> 4, l16 = lane & 15, t = l16 & 3, group = l16 >> 2;
  const int Hkv = a.num_kv_heads, h = wid % Hkv, b = blockIdx.y;
  const int pos0 = a.positions[b];
  if (pos0 < 0) {
    if (wid == 0 && lane == 0) report(a.status, DOE_DEVICE_ERR_PAGE);
    return;
  }
  const long long first = (long long)(pos0 & ~15) + 16ll * (wid / Hkv);
  const long long end = (long long)pos0 + a.n_tokens;
  if (first >= end) return;
  const int page = a.map.page(b, first);
  if (page < 0) {
    if (lane == 0) report(a.status, DOE_DEVICE_ERR_PAGE);
    return;
  }
  const int tiles = a.map.page_size / 16;
  const int tile = (int)(first % a.map.page_size) / 16;
  const size_t block = (((size_t)page * Hkv + h) * tiles + tile) * kI4Block;
  for (int kv = 0; kv < 2; ++kv) {
    const uint8_t* src = a.pool[kv] + block;
    T* dst = static_cast<T*>(a.out[kv]);
    uint32_t w[8];
    __half s[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int pair = 2 * j + hw;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (kv == 0) {
          const int tok = 2 * pair + e;
          w[2 * j + e] = *reinterpret_cast<const uint32_t*>(src + tok * 64 + t * 16 + group * 4);
          s[2 * j + e] = reinterpret_cast<const __half*>(src + kI4Codes)[tok * 4 + group];
        } else {
          w[2 * j + e] = *reinterpret_cast<const uint32_t*>(
              src + (((pair >> 2) * 8 + 2 * t + e) * 4 + (pair & 3)) * 16 + group * 4);
          s[2 * j + e] = reinterpret_cast<const __half*>(src + kI4Codes)[(pair * 4 + group) * 2 + e];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const long long pos = first + 2 * (2 * j + hw) + e;
        if (pos < pos0 || pos >= end) continue;
        const float sf = __half2float(s[2 * j + e]);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t n = kv == 0 ? (w[2 * j + e] >> (4 * (i >> 1) + 16 * (i & 1))) & 15u
                                     : (w[2 * j + (i >> 2)] >> (16 * e + 4 * (i & 3))) & 15u;
          v[i] = (float)((int)n - 8) * sf;
        }
        store8(dst + (((size_t)b * a.n_tokens + (size_t)(pos - pos0)) * Hkv + h) * 128 + 8 * l16, v);
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
  if (page < 0) {
    if (lane == 0) report(a.status, DOE_DEVICE_ERR_PAGE);
    return;
  }
  const int in_page = (int)(pos % a.map.page_size);
  const int Hkv = a.num_kv_heads, D = a.head_dim, n = Hkv * D;
  const size_t row = ((size_t)page * a.map.page_size + in_page) * n;
  const size_t out = ((size_t)b * a.n_tokens + tok) * n;
  for (int kv = 0; kv < 2; ++kv) {
    T* dst = static_cast<T*>(a.out[kv]) + out;
    for (int i = lane * 8; i < n; i += 256) {
      float v[8];
      if (INT8) {
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
    const uint64_t warps = (((uint64_t)a.n_tokens + 14) / 16 + 1) * kv->num_kv_heads;
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
