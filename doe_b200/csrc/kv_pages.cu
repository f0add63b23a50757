// kv_pages.cu -- copies of whole pages inside a paged KV cache: the device
// side of doe_kv_pool_make_writable (a shared page written by one of its
// sequences) and doe_kv_pool_compact.
//
// The page pairs come from the host's page pool, so they travel as kernel
// parameters: no staging buffer and no copy that the caller's list would have
// to outlive.  Bound by HBM: every page is read and written once.  8000 f16 pages of
// 64 KB take 169 us (6.2 TB/s, 0.95 of the measured copy rate), 8 int4 pages with
// their read-back 5 us: two launches.
#include "common.cuh"

namespace doe {

// Kernel parameters are limited to 32764 bytes; short lists take the small form
// because the parameters of every launch are copied.
template <int N>
struct PagePairs {
  int32_t page[2 * N];  // from, to
};

struct PageRegions {
  uint8_t* base[4];       // K, V and, for int8, their scales
  uint64_t page_bytes[2];  // of a K / V page, of a scale page (multiples of 16)
  uint32_t chunks[2];      // pieces of kPiece bytes per K / V page, per scale page
};

constexpr int kThreads = 256;
constexpr int kUnroll = 8;  // 16-byte loads in flight per thread (4: 188 us for 8000 f16 pages, 8: 180)
constexpr uint32_t kPiece = kThreads * kUnroll * 16;

// One CTA per (32 KB piece of a page, pair).
template <int N>
__global__ void __launch_bounds__(kThreads)
    copy_pages_kernel(const __grid_constant__ PagePairs<N> pairs, const PageRegions r) {
  pdl_wait();
  pdl_trigger();
  const uint32_t pair = blockIdx.y;
  const int32_t from = pairs.page[2 * pair], to = pairs.page[2 * pair + 1];
  uint32_t piece = blockIdx.x, region = 0;
  if (piece >= 2 * r.chunks[0]) {
    piece -= 2 * r.chunks[0];
    region = 2 + piece / r.chunks[1];
    piece %= r.chunks[1];
  } else {
    region = piece / r.chunks[0];
    piece %= r.chunks[0];
  }
  const uint64_t bytes = region < 2 ? r.page_bytes[0] : r.page_bytes[1];
  uint8_t* base = region == 0 ? r.base[0] : region == 1 ? r.base[1] : region == 2 ? r.base[2] : r.base[3];
  const uint4* src = reinterpret_cast<const uint4*>(base + (uint64_t)from * bytes);
  uint4* dst = reinterpret_cast<uint4*>(base + (uint64_t)to * bytes);
  const uint64_t n = bytes / 16, i0 = (uint64_t)piece * (kPiece / 16) + threadIdx.x;
  uint4 v[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u)
    if (i0 + u * kThreads < n) v[u] = __ldcs(src + i0 + u * kThreads);
#pragma unroll
  for (int u = 0; u < kUnroll; ++u)
    if (i0 + u * kThreads < n) dst[i0 + u * kThreads] = v[u];
}

template <int N>
static int launch_some(const int32_t* pairs, uint32_t n, const PageRegions& r, cudaStream_t st) {
  PagePairs<N> p;
  for (uint32_t i = 0; i < 2 * n; ++i) p.page[i] = pairs[i];
  const dim3 grid(2 * (r.chunks[0] + r.chunks[1]), n);
  return cuda_status(launch_pdl(copy_pages_kernel<N>, grid, dim3(kThreads), 0, st, p, r), "copy_pages_kernel");
}

int launch_copy_pages(const doe_paged_kv* kv, const int32_t* pairs, uint32_t n, const doe_launch* launch) {
  constexpr int kSmall = 60, kLarge = 4000;
  PageRegions r;
  const uint64_t rows = (uint64_t)kv->page_size * kv->num_kv_heads;
  r.base[0] = static_cast<uint8_t*>(kv->k_pool);
  r.base[1] = static_cast<uint8_t*>(kv->v_pool);
  r.base[2] = static_cast<uint8_t*>(kv->k_scale);
  r.base[3] = static_cast<uint8_t*>(kv->v_scale);
  r.page_bytes[0] = kv->kv_dtype == DOE_KV_F16    ? rows * kv->head_dim * 2
                    : kv->kv_dtype == DOE_KV_INT8 ? rows * kv->head_dim
                                                  : rows / 16 * DOE_KV_INT4_BLOCK_BYTES;
  r.page_bytes[1] = kv->kv_dtype == DOE_KV_INT8 ? rows * 2 : 0;
  for (int i = 0; i < 2; ++i) {
    const uint64_t c = (r.page_bytes[i] + kPiece - 1) / kPiece;
    if (c > 0x1fffffffull) {
      set_op_error("doe_paged_copy_pages: pages too large");
      return DOE_INVALID_ARGUMENT;
    }
    r.chunks[i] = (uint32_t)c;
  }
  cudaStream_t st = static_cast<cudaStream_t>(launch->stream);
  if (n <= kSmall) return launch_some<kSmall>(pairs, n, r, st);
  for (uint32_t i = 0; i < n; i += kLarge) {
    const int rc = launch_some<kLarge>(pairs + 2 * (size_t)i, n - i < kLarge ? n - i : kLarge, r, st);
    if (rc != DOE_OK) return rc;
  }
  return DOE_OK;
}

}  // namespace doe
