// logprobs.cu -- log probabilities of given tokens with the row's entropy and
// its top alternatives, over rows of logits (f32, f16 or bf16).
//
//   m = max x,  s = sum exp(x - m),  w = sum exp(x - m) (x - m)
//   logprob(t) = x_t - m - ln s,  entropy = ln s - w / s
// The exponent is (x - m) log2(e), rounded in that order: x log2(e) would
// overflow for logits masked with the type's lowest value.
//   top k by (value descending, index ascending); NaN orders as -inf
//
// One pass over the row: every element is loaded once, costs one exponential
// and a comparison with a threshold.  Bound by HBM for f32 and near the SFU's
// rate for 16-bit logits.  All sums are f32.
//
// Top k without sorting the row: the maxima of 32 disjoint thread groups are 32
// different elements, so their minimum is a value that at least 32 elements
// reach.  Elements below it are never candidates; the others (about 32 ln 32 of
// all those seen when it was taken) go into a shared buffer.  The threshold is
// renewed at the 1st, 2nd, 4th, 8th, ... step.  A full buffer (sorted or tied
// rows) is cut to its best k, whose last key then is the threshold.
//
// Few rows: a row is split over a cluster of up to 8 CTAs whose statistics and
// best k meet in the first CTA through distributed shared memory, so the call
// is one launch without workspace.
#include <cooperative_groups.h>

#include "common.cuh"

namespace doe {
namespace lp {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kCap = 2048;    // candidate buffer (a power of two)
constexpr int kUnroll = 4;    // 16-byte loads per thread and step
constexpr float kLn2 = 0.6931471805599453f;

struct Args {
  const void* logits;
  uint64_t row_stride;  // elements
  uint32_t vocab;
  uint32_t top_k;
  const int32_t* tokens;
  float* logprob;
  float* entropy;
  int32_t* top_ids;
  float* top_logprobs;
  int32_t* status;
};

// Order key: larger is better.  -0 counts as +0, NaN as -inf.
__device__ __forceinline__ unsigned long long key_of(float x, uint32_t index) {
  const uint32_t u = __float_as_uint(fmaxf(x, -INFINITY) + 0.0f);
  const uint32_t o = u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
  return ((unsigned long long)o << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ float value_of(unsigned long long key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
    x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
};
template <>
struct Vec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      x[2 * i] = f.x; x[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
};

// Running (m, s, w), w in log2 units; m = -inf: nothing but -inf seen.
struct Stat {
  float m, s, w;
};
__device__ __forceinline__ void raise(Stat& a, float m) {
  if (a.m == -INFINITY) {  // a.s counts only NaN so far
    a.w = a.s;
  } else {
    const float d = fmaxf((a.m - m) * kLog2e, -200.0f), c = ex2(d);  // 2^-200 is 0
    a.w = c * fmaf(d, a.s, a.w);
    a.s *= c;
  }
  a.m = m;
}
__device__ __forceinline__ Stat merge(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, a.s + b.s, a.w + b.w};
  if (a.m != m) raise(a, m);
  if (b.m != m) raise(b, m);
  return {m, a.s + b.s, a.w + b.w};
}

struct Shared {
  unsigned long long buf[kCap];
  unsigned long long sel[kMaxTop];  // the CTA's best k, in order
  unsigned long long thr_key;       // buffer cuts: only better keys matter
  float wmin[kWarps];
  Stat stat[kWarps];
  Stat total;
  uint32_t count;
};

// Sorts buf[0, n) descending; n is padded to a power of two with zeros.
__device__ void sort_keys(Shared& sh, uint32_t n) {
  uint32_t p = 2;
  while (p < n) p <<= 1;
  for (uint32_t i = n + threadIdx.x; i < p; i += kThreads) sh.buf[i] = 0;
  __syncthreads();
  for (uint32_t size = 2; size <= p; size <<= 1)
    for (uint32_t stride = size >> 1; stride > 0; stride >>= 1) {
      for (uint32_t i = threadIdx.x; i < p / 2; i += kThreads) {
        const uint32_t lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
        const bool down = (lo & size) == 0;
        const unsigned long long x = sh.buf[lo], y = sh.buf[hi];
        if ((x < y) == down) {
          sh.buf[lo] = y;
          sh.buf[hi] = x;
        }
      }
      __syncthreads();
    }
}

// The best k of buf[0, n) into sel, in order (zeros when n < k).  Ends synchronised.
__device__ void select(Shared& sh, uint32_t n, uint32_t k) {
  if (threadIdx.x < kMaxTop) sh.sel[threadIdx.x] = 0;
  __syncthreads();
  if (n <= kThreads) {  // keys differ, so a key's rank is the number of larger ones
    if (threadIdx.x < n) {
      const unsigned long long mine = sh.buf[threadIdx.x];
      uint32_t rank = 0;
      for (uint32_t i = 0; i < n; ++i) rank += sh.buf[i] > mine;
      if (rank < k) sh.sel[rank] = mine;
    }
  } else {
    sort_keys(sh, n);
    if (threadIdx.x < k) sh.sel[threadIdx.x] = sh.buf[threadIdx.x];
  }
  __syncthreads();
}

// A lower bound that at least 32 of the elements seen so far reach: the least
// of 32 groups' maxima (8 threads each).  Every thread gets it.
__device__ float group_bound(Shared& sh, float tmax) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) tmax = fmaxf(tmax, __shfl_xor_sync(0xffffffffu, tmax, o));
#pragma unroll
  for (int o = 8; o < 32; o <<= 1) tmax = fminf(tmax, __shfl_xor_sync(0xffffffffu, tmax, o));
  if ((threadIdx.x & 31) == 0) sh.wmin[threadIdx.x >> 5] = tmax;
  __syncthreads();
  float b = sh.wmin[0];
#pragma unroll
  for (int i = 1; i < kWarps; ++i) b = fminf(b, sh.wmin[i]);
  __syncthreads();
  return b;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const Args a, uint32_t splits) {
  __shared__ Shared sh;
  constexpr int N = Vec<T>::N;
  const uint32_t split = blockIdx.x, tid = threadIdx.x, k = a.top_k;
  const uint64_t row = blockIdx.y;
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  // 16-byte vectors from the row's base rounded down; the first and the last
  // may hold elements outside the row
  const uint32_t shift = (uint32_t)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const uint4* base = reinterpret_cast<const uint4*>(x - shift);
  const uint64_t nvec = ((uint64_t)shift + a.vocab + N - 1) / N;
  const uint64_t per = (nvec + splits - 1) / splits;
  const uint64_t v0 = split * per, v1 = v0 + per < nvec ? v0 + per : nvec;
  if (tid == 0) {
    sh.count = 0;
    sh.thr_key = 0;
  }
  __syncthreads();

  Stat st = {-INFINITY, 0.0f, 0.0f};
  float tmax = -INFINITY, bound = -INFINITY;
  uint32_t step = 0;
  for (uint64_t at = v0; at < v1; at += kThreads * kUnroll, ++step) {
    uint4 raw[kUnroll];
    float e[kUnroll][N];
    uint32_t live = 0;  // bit u: the vector holds elements of the row
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint64_t v = at + (uint64_t)u * kThreads + tid;
      if (v < v1 && (v > 0 || shift == 0) && (v + 1) * N <= (uint64_t)shift + a.vocab) {
        raw[u] = ldg_stream(base + v);
        live |= 1u << u;
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint64_t v = at + (uint64_t)u * kThreads + tid;
      if (live >> u & 1) {
        Vec<T>::unpack(raw[u], e[u]);
      } else if (v < v1) {  // an edge vector: elements outside the row count as absent (-inf)
        live |= 1u << u;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint64_t j = v * N + i;
          e[u][i] = j >= shift && j < (uint64_t)shift + a.vocab ? Vec<T>::one(x + (j - shift)) : -INFINITY;
        }
      }
    }
    float vmax = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (live >> u & 1)
#pragma unroll
        for (int i = 0; i < N; ++i) vmax = fmaxf(vmax, e[u][i]);
    if (vmax > st.m) raise(st, vmax);
    const float neg_m = st.m == -INFINITY ? 0.0f : -st.m;
    float2 s2 = make_float2(st.s, 0.0f), w2 = make_float2(st.w, 0.0f);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (live >> u & 1)
#pragma unroll
        for (int i = 0; i < N; i += 2) {
          const float2 d = fmul2(fadd2(make_float2(e[u][i], e[u][i + 1]), make_float2(neg_m, neg_m)),
                                 make_float2(kLog2e, kLog2e));
          const float2 p = make_float2(ex2(d.x), ex2(d.y));
          s2 = fadd2(s2, p);
          // clamped: a masked element adds 0 to w, not 0 * inf
          w2 = ffma2(p, make_float2(fmaxf(d.x, -200.0f), fmaxf(d.y, -200.0f)), w2);
        }
    st.s = s2.x + s2.y;
    st.w = w2.x + w2.y;
    if (k == 0) continue;
    tmax = fmaxf(tmax, vmax);
    if ((step & (step + 1)) == 0) bound = fmaxf(bound, group_bound(sh, tmax));
    // candidates; retried after a cut when the buffer was full
    unsigned long long pending = 0;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (live >> u & 1)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint64_t j = (at + (uint64_t)u * kThreads + tid) * N + i;
          if (!(e[u][i] < bound) && j >= shift && j < (uint64_t)shift + a.vocab) pending |= 1ull << (u * N + i);
        }
    while (true) {
      if (pending) {
        const unsigned long long thr = sh.thr_key;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (pending >> (u * N + i) & 1) {
              const uint64_t j = (at + (uint64_t)u * kThreads + tid) * N + i - shift;
              const unsigned long long key = key_of(e[u][i], (uint32_t)j);
              if (key <= thr) {
                pending &= ~(1ull << (u * N + i));
              } else {
                const uint32_t pos = atomicAdd(&sh.count, 1u);
                if (pos < kCap) {
                  sh.buf[pos] = key;
                  pending &= ~(1ull << (u * N + i));
                }
              }
            }
      }
      if (!__syncthreads_or(pending != 0)) break;
      // full: keep the best k; the last of them is the new threshold
      select(sh, kCap, k);
      if (tid < k) sh.buf[tid] = sh.sel[tid];
      if (tid == 0) {
        sh.count = k;
        sh.thr_key = sh.sel[k - 1];
      }
      bound = fmaxf(bound, value_of(sh.sel[k - 1]));
      __syncthreads();
    }
  }

  // ---- the CTA's statistics and best k -------------------------------------
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Stat b = {__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
                    __shfl_xor_sync(0xffffffffu, st.w, o)};
    st = merge(st, b);
  }
  if ((tid & 31) == 0) sh.stat[tid >> 5] = st;
  __syncthreads();
  if (tid == 0) {
    Stat t = sh.stat[0];
    for (int i = 1; i < kWarps; ++i) t = merge(t, sh.stat[i]);
    sh.total = t;
  }
  if (k != 0) {
    // drop what the last bound excludes, then order the rest
    bound = fmaxf(bound, group_bound(sh, tmax));
    const uint32_t n = sh.count;
    unsigned long long mine[kCap / kThreads];
#pragma unroll
    for (int i = 0; i < kCap / kThreads; ++i) mine[i] = i * kThreads + tid < n ? sh.buf[i * kThreads + tid] : 0;
    __syncthreads();
    if (tid == 0) sh.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kCap / kThreads; ++i)
      if (mine[i] != 0 && !(value_of(mine[i]) < bound)) sh.buf[atomicAdd(&sh.count, 1u)] = mine[i];
    __syncthreads();
    select(sh, sh.count, k);
  }
  if (splits > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (split == 0) {
      Stat t = sh.total;
      for (uint32_t i = 1; i < splits; ++i) t = merge(t, *cluster.map_shared_rank(&sh.total, i));
      unsigned long long key = 0;
      if (k != 0 && tid < splits * k) key = cluster.map_shared_rank(sh.sel, tid / k)[tid % k];
      __syncthreads();
      if (tid == 0) {
        sh.total = t;
        sh.count = 0;
      }
      __syncthreads();
      if (key != 0) sh.buf[atomicAdd(&sh.count, 1u)] = key;
      __syncthreads();
      if (k != 0) select(sh, sh.count, k);
    }
    cluster.sync();
    if (split != 0) return;
  }
  __syncthreads();
  const Stat t = sh.total;
  const bool none = t.s == 0.0f;  // every element is -inf
  const float ls = logf(t.s);
  if (tid == 0) {
    if (a.logprob != nullptr) {
      const int32_t token = a.tokens[row];
      float v = -INFINITY;
      if ((uint32_t)token < a.vocab)
        v = none ? -INFINITY : Vec<T>::one(x + token) - t.m - ls;
      else
        report(a.status, DOE_DEVICE_ERR_POSITION);
      a.logprob[row] = v;
    }
    if (a.entropy != nullptr) a.entropy[row] = none ? 0.0f : ls - t.w / t.s * kLn2;
  }
  if (tid < k) {
    const unsigned long long key = sh.sel[tid];
    a.top_ids[row * k + tid] = key != 0 ? (int32_t)(0xffffffffu - (uint32_t)key) : -1;
    a.top_logprobs[row * k + tid] = key == 0 || none ? -INFINITY : value_of(key) - t.m - ls;
  }
}

template <typename T>
int launch(const Args& a, uint64_t rows, cudaStream_t st) {
  // A row is split while the CTAs would leave SMs idle and every split still
  // has two steps' work.
  uint32_t splits = 1;
  const uint64_t step = (uint64_t)kThreads * kUnroll * Vec<T>::N;
  while (splits < 8 && rows * splits < 2ull * num_sms() && a.vocab > splits * step) splits *= 2;
  for (uint64_t r0 = 0; r0 < rows; r0 += 65535) {
    Args b = a;
    const uint64_t n = rows - r0 < 65535 ? rows - r0 : 65535;
    b.logits = static_cast<const T*>(a.logits) + r0 * a.row_stride;
    if (a.tokens) b.tokens = a.tokens + r0;
    if (a.logprob) b.logprob = a.logprob + r0;
    if (a.entropy) b.entropy = a.entropy + r0;
    if (a.top_ids) {
      b.top_ids = a.top_ids + r0 * a.top_k;
      b.top_logprobs = a.top_logprobs + r0 * a.top_k;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits, (unsigned)n);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const int rc = cuda_status(cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, b, splits), "logprobs_kernel");
    if (rc != DOE_OK) return rc;
  }
  return DOE_OK;
}

}  // namespace lp

int launch_token_logprobs(const void* logits, uint32_t dtype, uint64_t rows, uint32_t vocab, uint64_t row_stride,
                          const int32_t* tokens, uint32_t top_k, float* logprob, float* entropy, int32_t* top_ids,
                          float* top_logprobs, const doe_launch* launch) {
  lp::Args a;
  a.logits = logits;
  a.row_stride = row_stride;
  a.vocab = vocab;
  a.top_k = top_k;
  a.tokens = tokens;
  a.logprob = logprob;
  a.entropy = entropy;
  a.top_ids = top_ids;
  a.top_logprobs = top_logprobs;
  a.status = launch->status;
  cudaStream_t st = static_cast<cudaStream_t>(launch->stream);
  switch (dtype) {
    case DOE_DTYPE_F32: return lp::launch<float>(a, rows, st);
    case DOE_DTYPE_F16: return lp::launch<__half>(a, rows, st);
    default: return lp::launch<__nv_bfloat16>(a, rows, st);
  }
}

}  // namespace doe
