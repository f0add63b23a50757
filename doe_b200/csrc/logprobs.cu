// logprobs.cu -- log probabilities of given tokens with the row's entropy and
// its top alternatives, over rows of logits (f32, f16 or bf16).
//
//   m = max x,  s = sum exp(x - m),  w = sum exp(x - m) (x - m)
//   logprob(t) = x_t - m - ln s,  entropy = ln s - w / s
//   top k by (value descending, index ascending); NaN orders as -inf
//
// The exponent is one fma, x log2(e) - R with R = RN(m log2(e)), whose difference from
// (x - m) log2(e) is the same for the whole row and is taken off ln s at the end.  Where
// |m| is large, or x log2(e) overflows (rows of the type's lowest value), x - m comes
// first.  m is the warp's: it moves a few times a row, where a thread's own moved in
// nearly every step.  All sums are f32.
//
// One pass over the row: every element is loaded once, costs one exponential and a
// share of a maximum.  1024 rows of 128256 logits without alternatives take 49 us in
// bf16 (5.4 TB/s, 0.82 of the measured copy rate; the SFU's floor is 29), with 20 of
// them 70 us (0.57: barriers and candidates); f32 with 5 90 us (0.89).  64 rows of
// bf16 with 20 take 13.7 us, one row of 32000 5.4: launch, latency of the first loads
// and the joins.
//
// Loads go through a ring in shared memory (cp.async, every thread its own
// vectors, no barrier): 4 CTAs of 24 KB in flight per SM, where two vectors per
// thread in registers kept 24 KB and 0.54 of HBM.
//
// Top k without sorting the row: the maxima of 32 disjoint thread groups are 32
// different elements, so the k-th largest of them is a bound that at least k
// elements reach.  It is taken at the first step; elements above it go into a
// shared buffer.  After the 1st, 4th, 16th, ... step the buffer is cut to its
// best k, whose last value is the new bound: later elements equal to it lose by
// their index, so only larger ones matter, about k of them until the next cut.
// Between cuts the warps run on without a barrier (one per step cost 40 of 155 us
// at 1024 rows of 128256 bf16 logits), and a thread puts its own elements into the
// buffer (a scan over the warp for their places cost 19 of 96 us).  A row that fills the buffer all the same
// (rising ones, or a mask that leaves a group nothing) is gone over again with a cut
// whenever it is full; which of a step's elements fit is a matter of timing, so within
// the step the bound is the k-th one's value and index.  Where fewer
// than k elements lie above the first bound (rows that a mask or ties leave with
// few values) the first ones that equal it are looked for in another pass.
//
// Few rows: a row is split over a cluster of up to 8 CTAs, which write their
// statistics and best k into the first one's shared memory; it alone goes on (that
// it read theirs cost 1 us more).  So the call is one launch without workspace.
#include <cooperative_groups.h>

#include "common.cuh"

namespace doe {
namespace lp {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kMaxSplits = 8;
constexpr int kCap = 1024;    // candidate buffer (a power of two)
constexpr uint32_t kStages = 4;  // steps in the ring
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

// 16 bytes of logits: N elements.  Floor: what elements are raised to, see lowest().
template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4, kUnroll = 2;  // 16-byte loads per thread and step
  static constexpr uint32_t kLow = 0xff800000u;  // -inf
  static __device__ __forceinline__ float max(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static __device__ __forceinline__ float2 pair(const uint4& v, int i) {
    return i == 0 ? make_float2(__uint_as_float(v.x), __uint_as_float(v.y))
                  : make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  using Floor = float;
  static __device__ __forceinline__ Floor floor_of(float v) { return v; }
  static __device__ __forceinline__ float2 pair_over(const uint4& v, int i, Floor f) {
    const float2 x = pair(v, i);
    return make_float2(max_nan(x.x, f), max_nan(x.y, f));
  }
  // A bit per element above `bound`, and the element (of the thread's N kUnroll) of a bit.
  static __device__ __forceinline__ uint32_t above(const uint4 (&raw)[kUnroll], float bound) {
    uint32_t hits = 0;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const float2 f = pair(raw[u], i / 2);
        hits |= (f.x > bound ? 1u << (u * N + i) : 0u) | (f.y > bound ? 2u << (u * N + i) : 0u);
      }
    return hits;
  }
  static __device__ __forceinline__ uint32_t element(uint32_t bit) { return bit; }
};
__device__ __forceinline__ uint32_t word(const uint4& v, int i) {
  return i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w));
}
template <>
struct Vec<__half> {
  static constexpr int N = 8, kUnroll = 2;
  static constexpr uint32_t kLow = 0xfc00fc00u;
  static __device__ __forceinline__ float2 pair(const uint4& v, int i) {
    const uint32_t w = word(v, i);
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ float max(const uint4& v) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const float2 f = __half22float2(__hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3])));
    return fmaxf(f.x, f.y);
  }
  static __device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
  using Floor = __half2;
  static __device__ __forceinline__ Floor floor_of(float v) { return __half2half2(__float2half_rd(v)); }
  static __device__ __forceinline__ float2 pair_over(const uint4& v, int i, Floor f) {
    const uint32_t w = word(v, i);
    const __half2 x = __hmax2_nan(*reinterpret_cast<const __half2*>(&w), f);
    return __half22float2(x);
  }
  // `bound` is an element's value, so the conversion is exact; bits 0-15 are the words' low halves
  static __device__ __forceinline__ uint32_t above(const uint4 (&raw)[kUnroll], float bound) {
    const __half2 b = __float2half2_rn(bound);
    uint32_t hits = 0;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        hits |= __hgt2_mask(reinterpret_cast<const __half2*>(&raw[u])[i], b) & (0x00010001u << (4 * u + i));
    return hits;
  }
  static __device__ __forceinline__ uint32_t element(uint32_t bit) { return 2 * (bit & 15) + (bit >> 4); }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8, kUnroll = 2;
  static constexpr uint32_t kLow = 0xff80ff80u;
  static __device__ __forceinline__ float2 pair(const uint4& v, int i) {
    const uint32_t w = word(v, i);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ float max(const uint4& v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  using Floor = __nv_bfloat162;
  static __device__ __forceinline__ Floor floor_of(float v) { return __bfloat162bfloat162(__float2bfloat16_rd(v)); }
  static __device__ __forceinline__ float2 pair_over(const uint4& v, int i, Floor f) {
    const uint32_t w = word(v, i);
    const __nv_bfloat162 x = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w), f);
    return pair(make_uint4(*reinterpret_cast<const uint32_t*>(&x), 0, 0, 0), 0);
  }
  // `bound` is an element's value, so the conversion is exact; bits 0-15 are the words' low halves
  static __device__ __forceinline__ uint32_t above(const uint4 (&raw)[kUnroll], float bound) {
    const __nv_bfloat162 b = __float2bfloat162_rn(bound);
    uint32_t hits = 0;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        hits |= __hgt2_mask(reinterpret_cast<const __nv_bfloat162*>(&raw[u])[i], b) & (0x00010001u << (4 * u + i));
    return hits;
  }
  static __device__ __forceinline__ uint32_t element(uint32_t bit) { return 2 * (bit & 15) + (bit >> 4); }
};

// Running sums over elements x of d = (x - m) log2(e) + excess(m): s = sum 2^d and
// w = sum d 2^d.  m = -inf: nothing but -inf (and NaN, which s counts) seen.
struct Stat {
  float m, s, w;
};
// Up to this |m| the exponent is one fma, x log2(e) - R with R = m log2(e) rounded;
// its difference from (x - m) log2(e) is known.  Beyond, and for the type's lowest
// value, whose product overflows, x - m is taken first.
constexpr float kFused = 6e4f;  // lowest() is then above f16's lowest value, and excess() below 2^-8
__device__ __forceinline__ float excess(float m) { return fabsf(m) < kFused ? fmaf(m, kLog2e, -(m * kLog2e)) : 0.0f; }
// Elements below add nothing to sums over m; raised to this they add 0 d, not 0 * inf.
// Far enough below m in any of the types.
__device__ __forceinline__ float lowest(float m) { return m - fmaxf(150.0f, fabsf(m) * 0x1p-6f); }
__device__ __forceinline__ void raise(Stat& a, float m) {
  if (a.m == -INFINITY) {  // a.s counts only NaN so far
    a.w = a.s;
  } else {
    const float d = fmaxf(fmaf(a.m - m, kLog2e, excess(m) - excess(a.m)), -200.0f), c = ex2(d);  // 2^-200 is 0
    a.w = c * fmaf(d, a.s, a.w);
    a.s *= c;
  }
  a.m = m;
}
// Largest value of the warp's lanes.
__device__ __forceinline__ float redux_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;\n" : "=f"(r) : "f"(v));
  return r;
}
// The sum of all lanes' (a lane without one has {-inf, 0, 0}), on every lane.
__device__ __forceinline__ Stat warp_merge(Stat a) {
  const float m = redux_max(a.m);
  if (a.m != m) raise(a, m);
  return {m, warp_sum(a.s), warp_sum(a.w)};
}

struct Shared {
  alignas(16) unsigned long long buf[kCap];
  alignas(16) unsigned long long joined[kMaxSplits * kMaxTop];  // first CTA of a cluster: all CTAs' best k
  unsigned long long sel[kMaxTop];  // the CTA's best k, in order
  alignas(16) float group_max[32];
  float bound;
  Stat stat[kWarps];
  uint32_t hits[kWarps];
  Stat totals[kMaxSplits];  // first CTA of a cluster: of all CTAs
  uint32_t count;
  uint32_t full;  // candidates were lost
};

// Sorts buf[0, n) descending; n is padded to a power of two with zeros.
__device__ void sort_keys(unsigned long long* buf, uint32_t n) {
  uint32_t p = 2;
  while (p < n) p <<= 1;
  for (uint32_t i = n + threadIdx.x; i < p; i += kThreads) buf[i] = 0;
  __syncthreads();
  for (uint32_t size = 2; size <= p; size <<= 1)
    for (uint32_t stride = size >> 1; stride > 0; stride >>= 1) {
      for (uint32_t i = threadIdx.x; i < p / 2; i += kThreads) {
        const uint32_t lo = 2 * i - (i & (stride - 1)), hi = lo + stride;
        const bool down = (lo & size) == 0;
        const unsigned long long x = buf[lo], y = buf[hi];
        if ((x < y) == down) {
          buf[lo] = y;
          buf[hi] = x;
        }
      }
      __syncthreads();
    }
}

// The best k of buf[0, n), all different, into sel, in order (zeros when n < k).  buf
// has room for n rounded up to a power of two.  Ends synchronised.
__device__ void select(Shared& sh, unsigned long long* buf, uint32_t n, uint32_t k) {
  if (threadIdx.x >= n && threadIdx.x < k) sh.sel[threadIdx.x] = 0;
  if (n <= kThreads) {  // a key's rank is the number of larger ones
    if (threadIdx.x < n) {
      const unsigned long long mine = buf[threadIdx.x];
      uint32_t rank = 0;
      const ulonglong2* two = reinterpret_cast<const ulonglong2*>(buf);
#pragma unroll 8
      for (uint32_t i = 0; i < n / 2; ++i) rank += (two[i].x > mine) + (two[i].y > mine);
      if (n & 1) rank += buf[n - 1] > mine;
      if (rank < k) sh.sel[rank] = mine;
    }
  } else {
    sort_keys(buf, n);
    if (threadIdx.x < k) sh.sel[threadIdx.x] = buf[threadIdx.x];
  }
  __syncthreads();
}

// A lower bound that at least k of the elements seen so far reach: the k-th
// largest of 32 groups' maxima (8 threads each).  Every thread gets it.
__device__ float group_bound(Shared& sh, float tmax, uint32_t k) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) tmax = fmaxf(tmax, __shfl_xor_sync(0xffffffffu, tmax, o));
  if ((threadIdx.x & 7) == 0) sh.group_max[threadIdx.x >> 3] = tmax;
  __syncthreads();
  const uint32_t lane = threadIdx.x & 31;
  const float mine = sh.group_max[lane];
  uint32_t rank = 0;
#pragma unroll 8
  for (uint32_t i = 0; i < 32; ++i) {
    const float other = sh.group_max[i];
    rank += other > mine || (other == mine && i < lane);
  }
  const uint32_t at = __ballot_sync(0xffffffffu, rank == k - 1);
  const float bound = __shfl_sync(0xffffffffu, mine, __ffs(at) - 1);
  __syncthreads();
  return bound;
}

// Drops the candidates that are not above `bound`; the others stay, in any order.
// Synchronises before and after.
__device__ void filter(Shared& sh, float bound) {
  __syncthreads();
  const uint32_t n = min(sh.count, (uint32_t)kCap);
  unsigned long long mine[kCap / kThreads];
#pragma unroll
  for (int i = 0; i < kCap / kThreads; ++i) mine[i] = i * kThreads + threadIdx.x < n ? sh.buf[i * kThreads + threadIdx.x] : 0;
  __syncthreads();
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kCap / kThreads; ++i)
    if (mine[i] != 0 && value_of(mine[i]) > bound) sh.buf[atomicAdd(&sh.count, 1u)] = mine[i];
  __syncthreads();
}

// Keeps the best k of n >= k candidates; the last of them is the new bound.
__device__ void cut(Shared& sh, uint32_t n, uint32_t k, float& bound) {
  select(sh, sh.buf, n, k);
  if (threadIdx.x < k) sh.buf[threadIdx.x] = sh.sel[threadIdx.x];
  if (threadIdx.x == 0) sh.count = k;
  bound = fmaxf(bound, value_of(sh.sel[k - 1]));
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) logprobs_kernel(const Args a, uint32_t splits) {
  __shared__ Shared sh;
  __shared__ uint4 ring[kStages * Vec<T>::kUnroll * kThreads];  // every thread reads what it loaded
  using V = Vec<T>;
  constexpr int N = V::N, kUnroll = V::kUnroll;
  pdl_wait();
  pdl_trigger();
  const uint32_t split = blockIdx.x, tid = threadIdx.x, k = a.top_k;
  const uint64_t row = blockIdx.y;
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  // 16-byte vectors from the row's base rounded down; the first and the last
  // may hold elements outside the row, which count as -inf
  const uint32_t shift = (uint32_t)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const uint4* base = reinterpret_cast<const uint4*>(x - shift);
  const uint32_t nvec = (uint32_t)(((uint64_t)shift + a.vocab + N - 1) / N), per = (nvec + splits - 1) / splits;
  const uint32_t v0 = min(nvec, split * per), v1 = min(nvec, v0 + per);
  const uint32_t whole0 = shift ? 1 : 0, whole1 = (uint32_t)(((uint64_t)shift + a.vocab) / N);  // vectors within the row
  if (tid == 0) sh.count = sh.full = 0;
  Stat st = {-INFINITY, 0.0f, 0.0f};  // m is the warp's
  typename V::Floor floor = V::floor_of(0.0f);
  float tmax = -INFINITY, bound = -INFINITY;
  uint32_t step = 0;
  // This thread's elements above the bound (there are some) go into the buffer.  Their
  // values are read back from the ring's slot, where a run-time index costs nothing.
  // True: they did not all fit; none are taken, and their places stay empty.
  auto push = [&](const uint4 (&raw)[kUnroll], uint32_t at, uint32_t slot, float bound) {
    uint32_t hits = V::above(raw, bound), pos = atomicAdd(&sh.count, __popc(hits));
    const bool lost = pos + __popc(hits) > kCap;
    for (; hits != 0; hits &= hits - 1, ++pos) {
      const uint32_t e = V::element(__ffs(hits) - 1), u = e / N, i = e % N;
      const float v = V::one(reinterpret_cast<const T*>(&ring[(slot * kUnroll + u) * kThreads + tid]) + i);
      if (pos < kCap) sh.buf[pos] = lost ? 0ull : key_of(v, (at + u * kThreads + tid) * N + i - shift);
    }
    return lost;
  };
  // The same for elements whose key is above `kth`, of the step in slot 0.
  auto push_keys = [&](uint32_t at, unsigned long long kth) {
    constexpr uint32_t M = kUnroll * N;
    auto key_at = [&](uint32_t e) {
      const uint32_t u = e / N, i = e % N;
      const float v = V::one(reinterpret_cast<const T*>(&ring[u * kThreads + tid]) + i);
      return key_of(v, (at + u * kThreads + tid) * N + i - shift);
    };
    uint32_t n = 0;
#pragma unroll 1
    for (uint32_t e = 0; e < M; ++e) n += key_at(e) > kth;
    if (n == 0) return false;
    uint32_t pos = atomicAdd(&sh.count, n);
    const bool lost = pos + n > kCap;
#pragma unroll 1
    for (uint32_t e = 0; e < M; ++e) {
      const unsigned long long key = key_at(e);
      if (key <= kth) continue;
      if (pos < kCap) sh.buf[pos] = lost ? 0ull : key;
      ++pos;
    }
    return lost;
  };
  // An edge vector, element by element: those outside the row are -inf.
  auto edge = [&](uint32_t at, uint32_t slot, uint4 (&raw)[kUnroll]) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t v = at + u * kThreads + tid;
      if (v < v1 && (v < whole0 || v >= whole1)) {
        T e[N];
        uint4 low = make_uint4(V::kLow, V::kLow, V::kLow, V::kLow);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint64_t j = (uint64_t)v * N + i;
          e[i] = j >= shift && j < (uint64_t)shift + a.vocab ? x[j - shift] : reinterpret_cast<const T*>(&low)[i];
        }
        memcpy(&raw[u], e, 16);
        ring[(slot * kUnroll + u) * kThreads + tid] = raw[u];
      }
    }
  };
  constexpr uint32_t kStep = kThreads * kUnroll;  // vectors
  auto inside = [&](uint32_t v) { return v < v1 && v >= whole0 && v < whole1; };
  const uint32_t end = min(v1, whole1);
  auto all_inside = [&](uint32_t at) { return at >= whole0 && at + kStep <= end; };
  auto load = [&](uint32_t at, uint32_t slot) {
    const bool all = all_inside(at);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint32_t v = at + u * kThreads + tid;
      if (all || inside(v))
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(
                         (uint32_t)__cvta_generic_to_shared(&ring[(slot * kUnroll + u) * kThreads + tid])),
                     "l"(base + v)
                     : "memory");
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
#pragma unroll
  for (uint32_t i = 0; i < kStages - 1; ++i) load(v0 + i * kStep, i);
  if (splits > 1) cg::this_cluster().barrier_arrive();
  int32_t token = -1;
  float given = -INFINITY;  // the given token's logit
  if (split == 0 && tid == 0 && a.tokens != nullptr) {
    token = a.tokens[row];
    if ((uint32_t)token < a.vocab) given = V::one(x + token);
  }
  for (uint32_t at = v0; at < v1; at += kStep, ++step) {
    load(at + (kStages - 1) * kStep, (step + kStages - 1) % kStages);
    asm volatile("cp.async.wait_group %0;\n" ::"n"(kStages - 1) : "memory");
    uint4 raw[kUnroll];
    const uint32_t slot = step % kStages;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) raw[u] = ring[(slot * kUnroll + u) * kThreads + tid];
    if (!all_inside(at)) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (!inside(at + u * kThreads + tid)) raw[u] = make_uint4(V::kLow, V::kLow, V::kLow, V::kLow);
      edge(at, slot, raw);
    }
    float vmax = V::max(raw[0]);
#pragma unroll
    for (int u = 1; u < kUnroll; ++u) vmax = fmaxf(vmax, V::max(raw[u]));
    if (__any_sync(0xffffffffu, vmax > st.m)) {  // one m for the warp
      raise(st, redux_max(fmaxf(vmax, st.m)));
      floor = V::floor_of(lowest(st.m));
    }
    float2 s2 = make_float2(st.s, 0.0f), w2 = make_float2(st.w, 0.0f);
    if (fabsf(st.m) < kFused) {
      const float2 minus_r = make_float2(-(st.m * kLog2e), -(st.m * kLog2e));
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          const float2 d = ffma2(V::pair_over(raw[u], i, floor), make_float2(kLog2e, kLog2e), minus_r);
          const float2 p = make_float2(ex2(d.x), ex2(d.y));
          s2 = fadd2(s2, p);
          w2 = ffma2(p, d, w2);
        }
    } else {
      const float neg_m = st.m == -INFINITY ? 0.0f : -st.m;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
          const float2 d = fmul2(fadd2(V::pair(raw[u], i), make_float2(neg_m, neg_m)), make_float2(kLog2e, kLog2e));
          const float2 p = make_float2(ex2(d.x), ex2(d.y));
          s2 = fadd2(s2, p);
          w2 = ffma2(p, make_float2(fmaxf(d.x, -200.0f), fmaxf(d.y, -200.0f)), w2);
        }
    }
    st.s = s2.x + s2.y;
    st.w = w2.x + w2.y;
    if (k == 0) continue;
    tmax = fmaxf(tmax, vmax);
    if (step == 0) bound = group_bound(sh, tmax, k);
    if (vmax > bound && push(raw, at, slot, bound)) sh.full = 1;
    // 1st, 4th, 16th, ... step, but not the last
    if ((step & (step + 1)) == 0 && (step + 1 & 0x55555555u) != 0 && at + kStep < v1) {
      __syncthreads();
      const uint32_t n = sh.count;
      if (n > k && sh.full == 0) cut(sh, n, k, bound);
      else __syncthreads();  // before the next candidates are counted
    }
  }
  st.s = warp_sum(st.s);
  st.w = warp_sum(st.w);
  if ((tid & 31) == 0) sh.stat[tid >> 5] = st;
  __syncthreads();
  if (k != 0 && sh.full) {
    __syncthreads();
    if (tid == 0) sh.count = 0;
    bound = tmax = -INFINITY;
    for (uint32_t at = v0; at < v1; at += kStep) {
      uint4 raw[kUnroll];
      float vmax = -INFINITY;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        raw[u] = make_uint4(V::kLow, V::kLow, V::kLow, V::kLow);
        if (inside(at + u * kThreads + tid)) raw[u] = __ldcs(base + at + u * kThreads + tid);
        ring[u * kThreads + tid] = raw[u];
      }
      if (at < whole0 || at + kStep > whole1) edge(at, 0, raw);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) vmax = fmaxf(vmax, V::max(raw[u]));
      tmax = fmaxf(tmax, vmax);
      if (at == v0) bound = group_bound(sh, tmax, k);
      bool todo = true;
      unsigned long long kth = 0;
      for (int round = 0;; ++round) {
        todo = todo && (kth == 0 ? vmax > bound && push(raw, at, 0, bound) : vmax >= bound && push_keys(at, kth));
        if (!__syncthreads_or(todo)) break;
        if (round == 0) {  // a new bound
          bound = fmaxf(bound, group_bound(sh, tmax, k));
          filter(sh, bound);
        } else {
          // full again: the best k so far are the bound, for the rest of this step by value and
          // index, as elements left out may come before kept ones that they equal
          cut(sh, kCap, k, bound);
          kth = sh.sel[k - 1];
        }
      }
    }
  }

  // ---- the CTA's statistics and best k -------------------------------------
  if (tid >= kThreads - 32) {  // the warp that select() needs least
    const uint32_t lane = tid & 31;
    st = warp_merge(lane < kWarps ? sh.stat[lane] : Stat{-INFINITY, 0.0f, 0.0f});
    if (lane == 0) sh.totals[0] = st;
  }
  if (k != 0) {
    uint32_t n = sh.count;
    select(sh, sh.buf, n, k);
    if (n < k) {
      // the rest are the first elements that equal the bound (a NaN equals -inf)
      const uint64_t j1 = min((uint64_t)a.vocab, max((uint64_t)v1 * N, (uint64_t)shift) - shift);
      for (uint64_t j0 = max((uint64_t)v0 * N, (uint64_t)shift) - shift; j0 < j1 && n < k; j0 += kThreads) {
        const uint64_t j = j0 + tid;
        float v = 0.0f;
        bool equal = false;
        if (j < j1) {
          v = V::one(x + j);
          equal = bound == -INFINITY ? !(v > bound) : v == bound;
        }
        const uint32_t mask = __ballot_sync(0xffffffffu, equal);
        if ((tid & 31) == 0) sh.hits[tid >> 5] = __popc(mask);
        __syncthreads();
        uint32_t pos = n + __popc(mask & ((1u << (tid & 31)) - 1));
        for (uint32_t w = 0; w < kWarps; ++w) {
          if (w < tid >> 5) pos += sh.hits[w];
          n += sh.hits[w];
        }
        if (equal && pos < k) sh.sel[pos] = key_of(v, (uint32_t)j);
        __syncthreads();
      }
    }
  }
  if (splits > 1) {
    // every CTA writes into the first one's shared memory, which none of them reads after
    // it has gone
    cg::cluster_group cluster = cg::this_cluster();
    Shared* first = cluster.map_shared_rank(&sh, 0);
    if (k == 0) __syncthreads();  // totals[0]; select() ends with one
    const Stat mine = sh.totals[0];
    cluster.barrier_wait();  // the first CTA runs, and has not yet reached the next sync
    // entries without an element differ too; their upper half is 0
    if (tid < k) first->joined[split * k + tid] = sh.sel[tid] != 0 ? sh.sel[tid] : split * k + tid + 1;
    if (tid == 0 && split != 0) first->totals[split] = mine;
    cluster.sync();
    if (split != 0) return;
    if (tid >= kThreads - 32) {
      const uint32_t lane = tid & 31;
      st = warp_merge(lane < splits ? sh.totals[lane] : Stat{-INFINITY, 0.0f, 0.0f});
      if (lane == 0) sh.totals[0] = st;
    }
    if (k != 0) select(sh, sh.joined, splits * k, k);
  }
  if (k == 0) __syncthreads();
  const Stat t = sh.totals[0];
  const bool none = t.s == 0.0f;  // every element is -inf
  const float log2s = log2f(t.s), ls = (log2s - excess(t.m)) * kLn2;
  if (tid == 0) {
    if (a.logprob != nullptr) {
      if ((uint32_t)token >= a.vocab) report(a.status, DOE_DEVICE_ERR_POSITION);
      a.logprob[row] = none || (uint32_t)token >= a.vocab ? -INFINITY : given - t.m - ls;
    }
    if (a.entropy != nullptr) a.entropy[row] = none ? 0.0f : (log2s - t.w / t.s) * kLn2;
  }
  if (tid < k) {
    const unsigned long long key = sh.sel[tid];
    const bool some = key >> 32 != 0;
    a.top_ids[row * k + tid] = some ? (int32_t)(0xffffffffu - (uint32_t)key) : -1;
    a.top_logprobs[row * k + tid] = !some || none ? -INFINITY : value_of(key) - t.m - ls;
  }
}

template <typename T>
int launch(const Args& a, uint64_t rows, cudaStream_t st) {
  // A row is split while there are at most 3 CTAs per SM (4 are resident; a split costs
  // its own cuts: 64 rows of 128257 bf16 logits in 4 splits 15.6 us, in 8 18.7, in 2 23.5) and every split
  // still has two steps' work.
  uint32_t splits = 1;
  const uint64_t step = (uint64_t)kThreads * Vec<T>::kUnroll * Vec<T>::N;
  while (splits < (uint32_t)kMaxSplits && rows * splits * 2 <= 3ull * num_sms() && a.vocab > splits * step) splits *= 2;
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
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = splits;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = splits > 1 ? 2 : 1;
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
