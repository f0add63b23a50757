// paged_decode_int4.cu -- batched GQA decode over the 4-bit paged KV cache
// (int4.cuh), split over the KV length, with the fused new-token append.
//
// Semantics: those of paged_decode.cu (one query per sequence, GQA, window,
// softcap, RoPE, out = acc / l or 0 when l == 0) on the values (n - 8) * s of
// the cache.  1 to 8 query heads per kv head.
//
// Mathematics.  With K codes n and scales s[token][group],
//   S[token, head] = sum_group s * (sum_{d in group} n q - 8 sum_{d in group} q)
//   O[dim, head]   = sum_token (n - 8) (s[token][group(dim)] p[token, head])
// Both products run on mma.sync m16n8k16 with the codes as the A operand and
// the (up to 8) heads as its 8 columns: S = K Q^T takes 16 tokens as rows, O^T =
// V^T P^T 16 dims.  A code pair masked out of its word, (w >> 4 i) &
// 0x000f000f, IS an f16 pair: the subnormals n * 2^-24, exact in the tensor
// core; the pair at bits 4-7 is left there and reads n * 2^-20.  So 8 codes cost
// one shift and 4 ANDs.  The powers of two go into Q (words of the high
// nibbles times 2^-4), the score scale (2^24) and the final accumulators; -8
// becomes the S accumulators' start value (-8 sum q) and, for O, one MMA per
// group with a constant A operand (8) on the same B operand, so exactly the
// f16 (s p) the product used is taken off.
// P moves from the S accumulators (token rows) into the B operand (head
// columns) by movmatrix.  S, the softmax statistics and O are f32; P and s p are
// rounded to f16 (2^-12 relative, the f16 and int8 kernels' choice).
//
// The running reference of a head, m, is its score maximum plus the exponent
// of the V scales seen, so that s p stays within f16's range and out of its
// subnormals whatever the magnitude of V.  It is lazy: it moves only when a
// score exceeds it by 2^8 or a V scale exceeds the exponent.
//
// Loads: a warp walks its blocks kStep at a time out of a ring of its own in
// shared memory, filled with cp.async: a block is 1024 + 128 contiguous bytes
// of K and of V, 5 instructions for the warp.  (One elected lane issuing two
// bulk copies costs the warp some 45 instructions, waits included, of about 270
// a block: 128 us for 64 sequences of 1k-8k tokens.)
//
// Work: see plan().  Many rows (sequence, kv head): the blocks of all of them are
// one list that the resident CTAs share out evenly, so that ragged lengths leave
// no tail; a row that a share's end cuts is stitched by the last of its CTAs to
// arrive.  Few rows: each is cut into splits of one length, up to 8 of which form
// a cluster and join in distributed shared memory, each CTA a slice of the dims;
// the clusters are stitched per slice by the last one to arrive.  Sums go in the
// order of the keys, so results do not depend on timing.
#include <cooperative_groups.h>
#include <cstdlib>

#include "int4.cuh"

namespace doe {
namespace i4 {

namespace cg = cooperative_groups;

constexpr int kD = 128;
constexpr int kWarps = 4;
#ifndef I4STEP
#define I4STEP 2
#define I4OCC 3
#define I4STAGES 6
#endif
constexpr int kStep = I4STEP;                       // blocks per loop step
constexpr int kStages = I4STAGES;                     // ring slots, a multiple of kStep
constexpr int kBlkRing = 128;                  // block numbers per warp, renewed 32 at a time
constexpr int kCtasPerSm = I4OCC;                  // resident: 168 registers a thread
constexpr uint32_t kMaxStreamSeqs = 1024;      // sequences whose lengths a CTA adds up
constexpr int kSlot = 2 * kI4Block;            // K block, V block
constexpr int kWarpBytes = kStages * kSlot;    // also holds the warp's O, 8 x 128 f32
constexpr int kSmem = kWarps * kWarpBytes;
static_assert(kWarpBytes >= 8 * kD * 4, "the merge stages a warp's O in its ring");

struct Args {
  const __half* q;  // [B, H, 128]
  uint8_t* k_pool;  // blocks [num_pages, Hkv, page_size / 16]
  uint8_t* v_pool;
  const int32_t* block_table;
  const int32_t* seq_lens;
  const __half* new_k;  // [B, Hkv, 128] or null
  const __half* new_v;
  float* out;           // [B, H, 128] f32, or bf16 storage when out_bf16
  float* part_o;        // splits: [B * Hkv * max_parts, group, 128]; shares: [CTAs, 2, group, 128]
  float* part_ml;       // [.., slices, group, 2] / [.., group, 2]
  unsigned* counters;   // [B * Hkv, slices], zero at launch, left zero by the stitch
  int32_t* status;
  const float* freq_cis;
  int rope_positions;
  int window;
  float softcap;
  float scale;
  int num_heads, num_kv_heads, group, num_pages, page_size, max_pages;
  int tiles_per_page, tile_shift;  // page_size / 16 and its log2 (-1: not a power of two)
  int num_seqs;
  int split_tiles, max_parts;  // splits: blocks per split, clusters (or single splits) per row
  int out_bf16;
  int inputs_stable;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes, or zeros when size is 0
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t size) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(size) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}
// mma_16816 with a start value apart from the result
__device__ __forceinline__ void mma_from(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1, float c0, float c1, float c2, float c3) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) {
  return i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w));
}
// 8x8 transpose of 16-bit elements across the warp: lane 4 i + j gives
// (row i, cols 2 j, 2 j + 1) and gets them of the transpose.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hmax2(uint32_t a, uint32_t b) {
  const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float2 f2(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

// The new token's row of kv head g, written by one warp: load() right after
// the launch's wait, store() once the loads have landed.  Lane l owns dims
// [4 l, 4 l + 4): half of a K word, one 16-bit half of the V block.
struct AppendRow {
  uint2 raw[2];
  float rc[4], rsn[4];
  int page, tile, tok;

  __device__ __forceinline__ void load(const Args& a, int b, int g, int pos, const int32_t* table, int lane) {
    const int pidx = pos / a.page_size, in_page = pos - pidx * a.page_size;
    page = table[pidx];
    tile = in_page >> 4;
    tok = in_page & 15;
    const size_t src = ((size_t)b * a.num_kv_heads + g) * kD + 4 * lane;
    raw[0] = *reinterpret_cast<const uint2*>(a.new_k + src);
    raw[1] = *reinterpret_cast<const uint2*>(a.new_v + src);
    if (a.freq_cis != nullptr)
      rope_table<2>(a.freq_cis, a.rope_positions, kD / 2, pos, 4 * (lane & 15), a.status, lane == 0, rc, rsn);
  }

  // Ends with the barrier that lets the warp's later copies read the row.
  __device__ __forceinline__ void store(const Args& a, int g, int lane) {
    if ((unsigned)page >= (unsigned)a.num_pages) {
      if (lane == 0) report(a.status, DOE_DEVICE_ERR_PAGE);
      return;
    }
    const size_t block = (((size_t)page * a.num_kv_heads + g) * a.tiles_per_page + tile) * kI4Block;
    const int group = lane >> 3;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      uint2 v = raw[kv];
      if (kv == 0 && a.freq_cis != nullptr) {
        const uint2 p = make_uint2(__shfl_xor_sync(0xffffffffu, v.x, 16), __shfl_xor_sync(0xffffffffu, v.y, 16));
        rope_rotate<2>(reinterpret_cast<const uint32_t*>(&raw[0]), reinterpret_cast<const uint32_t*>(&p), lane < 16,
                       rc, rsn, reinterpret_cast<uint32_t*>(&v));
      }
      const float2 x01 = f2(v.x), x23 = f2(v.y);
      float amax = fmaxf(fmaxf(fabsf(x01.x), fabsf(x01.y)), fmaxf(fabsf(x23.x), fabsf(x23.y)));
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const __half sh = __float2half_rn(div7(amax));
      const float s = __half2float(sh);
      const float rs = s != 0.0f ? __frcp_rn(s) : 0.0f;
      uint32_t c[4] = {8u, 8u, 8u, 8u};
      if (s != 0.0f) {
        c[0] = quantize_u4(x01.x, s, rs);
        c[1] = quantize_u4(x01.y, s, rs);
        c[2] = quantize_u4(x23.x, s, rs);
        c[3] = quantize_u4(x23.y, s, rs);
      }
      uint8_t* dst = (kv ? a.v_pool : a.k_pool) + block;
      if (kv == 0) {
        // even lanes hold dims 0..3 of the word's 8, odd lanes dims 4..7
        uint32_t w = (c[0] | (c[1] << 16) | (c[2] << 4) | (c[3] << 20)) << (8 * (lane & 1));
        w |= __shfl_xor_sync(0xffffffffu, w, 1);
        if ((lane & 1) == 0) *reinterpret_cast<uint32_t*>(dst + tok * 64 + ((lane & 7) >> 1) * 16 + group * 4) = w;
        if ((lane & 7) == 0) *reinterpret_cast<__half*>(dst + kI4Codes + (tok * 4 + group) * 2) = sh;
      } else {
        const uint32_t w = c[0] | (c[1] << 4) | (c[2] << 8) | (c[3] << 12);
        *reinterpret_cast<uint16_t*>(dst + (((tok >> 3) * 8 + (lane & 7)) * 4 + ((tok >> 1) & 3)) * 16 + group * 4 +
                                     2 * (tok & 1)) = (uint16_t)w;
        if ((lane & 7) == 0)
          *reinterpret_cast<__half*>(dst + kI4Codes + (((tok >> 1) * 4 + group) * 2 + (tok & 1)) * 2) = sh;
      }
    }
    __threadfence_block();
    __syncwarp();
  }
};

constexpr int kDead = -1, kMasked = (int)0x80000000u;  // of a block number
constexpr float kNone = -1e30f;  // the reference of a head without keys: below any score
constexpr uint32_t kLo = 0x000f000fu, kHi = 0x00f000f0u, kBoth = 0x00ff00ffu;
constexpr float kTwo24 = 16777216.0f;

// One sequence's keys: [min_key, seq_len), in blocks from `origin` on.
struct Keys {
  int seq_len, min_key, origin, tiles;
};
__device__ __forceinline__ Keys keys_of(const Args& a, int raw_len) {
  Keys s;
  const int cap = a.max_pages * a.page_size;
  s.seq_len = raw_len < 0 ? 0 : (raw_len > cap ? cap : raw_len);
  // the window's keys; the walk starts at the block holding the first
  s.min_key = (a.window > 0 && s.seq_len > a.window) ? s.seq_len - a.window : 0;
  s.origin = s.min_key >> 4;
  s.tiles = ((s.seq_len + 15) >> 4) - s.origin;
  return s;
}

// Even shares of a list: `size` entries each, one more in the first `more`.
struct Share {
  int size, more;
  __device__ __forceinline__ int begin(int c) const { return c * size + min(c, more); }
  __device__ __forceinline__ int owner(int x) const {
    const int cut = more * (size + 1);
    return x < cut ? x / (size + 1) : more + (x - cut) / size;
  }
};

// SHARES: the CTA's share of the list of all blocks; else one split of one row.
template <bool CAP, bool SHARES>
__global__ void __launch_bounds__(kWarps * 32, kCtasPerSm) decode_kernel(const Args a) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float sm_m[kWarps][8];
  __shared__ float sm_l[kWarps][8];
  __shared__ float cta_ml[8][2];
  __shared__ int sm_last;
  __shared__ __align__(8) int sm_blk[kWarps][kBlkRing];
  __shared__ int sm_end[SHARES ? kMaxStreamSeqs : 1];  // blocks of sequences 0..b (one kv head)
  __shared__ int sm_sum[kWarps];

  if (!a.inputs_stable) pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, t = lane & 3;
  const int Hkv = a.num_kv_heads, group = a.group;
  const int slices = SHARES ? 1 : (int)cg::this_cluster().num_blocks();

  // ---- what this CTA walks ------------------------------------------------------
  Share share = {};
  int at = 0, end = 0, b = 0;  // SHARES: [at, end) of the list, Hkv rows per sequence
  if (SHARES) {
    // running sum of the sequences' blocks; an empty one counts as a block, so
    // that a CTA writes its zeros
    const int per = (a.num_seqs + kWarps * 32 - 1) / (kWarps * 32), b0 = threadIdx.x * per;
    int sum = 0;
    for (int i = b0; i < min(b0 + per, a.num_seqs); ++i) {
      const int raw = a.seq_lens[i];
      const Keys s = keys_of(a, raw);
      if (raw != s.seq_len && blockIdx.x == 0) report(a.status, DOE_DEVICE_ERR_LENGTH);
      sum += max(1, s.tiles);
      sm_end[i] = sum;
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) sm_sum[warp] = incl;
    __syncthreads();
    int before = incl - sum;
    for (int w = 0; w < warp; ++w) before += sm_sum[w];
    for (int i = b0; i < min(b0 + per, a.num_seqs); ++i) sm_end[i] += before;
    __syncthreads();
    const int total = sm_end[a.num_seqs - 1] * Hkv;  // below 2^31 (plan)
    // at least two blocks per warp and share, unless there are more rows
    const int shares = min((int)gridDim.x, max(total / (2 * kWarps), a.num_seqs * Hkv));
    if ((int)blockIdx.x >= shares) return;
    share.size = total / shares;
    share.more = total - share.size * shares;
    at = share.begin(blockIdx.x);
    end = share.begin(blockIdx.x + 1);
    int hi = a.num_seqs - 1;  // the first sequence that ends after `at`
    while (b < hi) {
      const int mid = (b + hi) >> 1;
      if (sm_end[mid] * Hkv > at) hi = mid;
      else b = mid + 1;
    }
  }
  for (bool first_row = true;; first_row = false) {
  int g, tile_begin, tile_end, part = 0, nparts;
  Keys seq;
  size_t row;
  int row_at = 0;
  if (SHARES) {
    if (at >= end) break;
    if (!first_row) {
      __syncthreads();  // the last row's staging and statistics have been read
      if (at >= sm_end[b] * Hkv) ++b;
    }
    const int seq_at = b ? sm_end[b - 1] : 0, size = sm_end[b] - seq_at;
    g = (at - seq_at * Hkv) / size;
    row_at = seq_at * Hkv + g * size;
    seq = keys_of(a, a.seq_lens[b]);
    tile_begin = at - row_at;
    tile_end = min(end - row_at, size);
    at = row_at + tile_end;
    nparts = tile_begin == 0 && tile_end == size ? 1 : 2;  // the exact number where it matters
    tile_end = min(tile_end, seq.tiles);
  } else {
    g = blockIdx.y;
    b = blockIdx.z;
    const int raw = a.seq_lens[b], split = blockIdx.x;
    seq = keys_of(a, raw);
    if (raw != seq.seq_len && split == 0 && g == 0 && threadIdx.x == 0) report(a.status, DOE_DEVICE_ERR_LENGTH);
    const int nsplits = max(1, (seq.tiles + a.split_tiles - 1) / a.split_tiles);
    part = split / slices;
    nparts = nsplits == 1 ? 0 : (nsplits + slices - 1) / slices;  // 0: nothing to join, not even in the cluster
    if (split >= max(nparts, 1) * slices) return;  // the whole cluster; a split past the last joins with nothing
    if (nparts == 0 && split != 0) return;
    tile_begin = split * a.split_tiles;
    tile_end = min(seq.tiles, tile_begin + a.split_tiles);
  }
  row = (size_t)b * Hkv + g;
  const int seq_len = seq.seq_len, min_key = seq.min_key;
  const int32_t* table = a.block_table + (size_t)b * a.max_pages;

  // this warp's blocks: first + kWarps * k, k < nt, as block numbers in the pools,
  // looked up 96 ahead.  kDead: past the walk, or on a page outside the pool;
  // kMasked is set on a block with dead keys (the window's first, the sequence's
  // last)
  const int first = seq.origin + tile_begin + warp;
  const int span = tile_end - tile_begin - warp;
  const int nt = span > 0 ? (span + kWarps - 1) / kWarps : 0;
  auto block_number = [&](int i) {
    if (i >= nt) return kDead;
    const int tile = first + kWarps * i;
    const int pidx = a.tile_shift >= 0 ? tile >> a.tile_shift : tile / a.tiles_per_page;
    const int page = table[pidx];
    if ((unsigned)page < (unsigned)a.num_pages)
      return (page * Hkv + g) * a.tiles_per_page + (tile - pidx * a.tiles_per_page) +
             (tile * 16 < min_key || tile * 16 + 16 > seq_len ? kMasked : 0);
    report(a.status, DOE_DEVICE_ERR_PAGE);
    return kDead;
  };
#pragma unroll
  for (int i = 0; i < kBlkRing - 32; i += 32) sm_blk[warp][i + lane] = i < nt + kStages ? block_number(i + lane) : kDead;
  int ahead = nt > kBlkRing - 32 ? block_number(kBlkRing - 32 + lane) : kDead;
  __syncwarp();

  const uint32_t wbase = smem_addr(ring) + warp * kWarpBytes;
  const uint8_t* k_lane = a.k_pool + 16 * lane;
  const uint8_t* v_lane = a.v_pool + 16 * lane;
  // lanes 0-7 copy the K scales, 8-15 the V scales
  const uint8_t* s_lane = (lane < 8 ? k_lane : v_lane - 128) + kI4Codes;
  const uint32_t lane_dst = wbase + 16 * lane;
  const uint32_t s_dst = lane_dst + kI4Codes + (lane < 8 ? 0 : kI4Block - 128);
  // Fills the slot at byte `slot` of the ring with block number blk, a dead one
  // with zeros
  auto issue = [&](int blk, uint32_t slot) {
    const uint32_t size = blk == kDead ? 0u : 16u;
    const size_t off = (size_t)(blk == kDead ? 0u : (uint32_t)blk & ~(uint32_t)kMasked) * kI4Block;
    copy16(lane_dst + slot, k_lane + off, size);
    copy16(lane_dst + slot + 512, k_lane + off + 512, size);
    copy16(lane_dst + slot + kI4Block, v_lane + off, size);
    copy16(lane_dst + slot + kI4Block + 512, v_lane + off + 512, size);
    if (lane < 16) copy16(s_dst + slot, s_lane + off, size);
  };

  // first copies before the query work (and before griddepcontrol.wait when the
  // caller vouches for the inputs); the block that receives the new row, the walk's
  // last of the warp that appends it, waits for the append
  const bool append_pending =
      a.new_k != nullptr && seq_len > 0 && nt > 0 && first + kWarps * (nt - 1) == (seq_len - 1) >> 4;
  const int early = min(kStages - kStep, append_pending ? nt - 1 : nt);
  for (int k = 0; k < early; ++k) {
    issue(sm_blk[warp][k], k * kSlot);
    if (k % kStep == kStep - 1) copy_commit();
  }
  if (first_row) {
    if (a.inputs_stable) pdl_wait();
    pdl_trigger();
  }
  AppendRow app;
  if (append_pending) app.load(a, b, g, seq_len - 1, table, lane);

  // ---- Q as the B operand: lane (r = head, t) holds dims 32 grp + 8 t + 0..7,
  // word i of each run = dims (2 i, 2 i + 1) = the K word's nibbles i and i + 4
  uint32_t qb[4][4];
  float qinit[4][4];  // -8 sum_group q of heads 2 t, 2 t + 1 (times 2^-24), for both token rows
  {
    const __half* qrow = a.q + ((size_t)b * a.num_heads + (size_t)g * group + r) * kD;
    const bool live = r < group;
    uint4 qv[4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
      qv[n] = live ? *reinterpret_cast<const uint4*>(qrow + 32 * n + 8 * t) : make_uint4(0, 0, 0, 0);
    if (a.freq_cis != nullptr && live && seq_len > 0) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        float rc[8], rsn[8];
        rope_table<4>(a.freq_cis, a.rope_positions, kD / 2, (long long)seq_len - 1, 32 * n + 8 * t, a.status,
                      tile_begin == 0 && g == 0 && lane == 0 && warp == 0, rc, rsn);
        const uint4 lo = qv[n], hi = qv[n + 2];
        rope_rotate<4>(reinterpret_cast<const uint32_t*>(&lo), reinterpret_cast<const uint32_t*>(&hi), true, rc, rsn,
                       reinterpret_cast<uint32_t*>(&qv[n]));
        rope_rotate<4>(reinterpret_cast<const uint32_t*>(&hi), reinterpret_cast<const uint32_t*>(&lo), false, rc, rsn,
                       reinterpret_cast<uint32_t*>(&qv[n + 2]));
      }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      float qs = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w = word(qv[n], i) ^ (!CAP && a.scale < 0.0f ? 0x80008000u : 0u);
        float mult = 1.0f;
        if (i & 1) {  // meets codes read as n 2^-20; q 2^-4 loses bits only below |q| = 2^-10, 2^-21 absolute
          w = hmul2(w, 0x2c002c00u);
          mult = 16.0f;
        }
        qb[n][i] = w;
        const float2 f = f2(w);
        qs += mult * (f.x + f.y);
      }
      qs += __shfl_xor_sync(0xffffffffu, qs, 1);
      qs += __shfl_xor_sync(0xffffffffu, qs, 2);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        qinit[n][j] = -8.0f / kTwo24 * __shfl_sync(0xffffffffu, qs, (2 * t + j) * 4);
        qinit[n][2 + j] = qinit[n][j];
        asm("" : "+f"(qinit[n][2 + j]));  // a quad of registers of its own: the MMA takes it without copies
      }
    }
  }

  // heads 2 t and 2 t + 1 of this lane's accumulator columns
  float m_ref[2] = {kNone, kNone}, l_run[2] = {0.0f, 0.0f};
  int v_exp = -3;                // every V scale seen is at most 2^v_exp (or infinite)
  uint32_t v_lim = 0x30003000u;  // 2^v_exp as an f16 pair
  float m_lim[2] = {kNone, kNone};  // x of a score 2^8 over its maximum
  float acc[8][4], off[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;

  if (append_pending) app.store(a, g, lane);
  for (int k = early; k < kStages - kStep; ++k) {
    issue(sm_blk[warp][k], k * kSlot);
    if (k % kStep == kStep - 1) copy_commit();
  }

  // x is the softcapped score in the log2 domain (CAP) or the bare product, which
  // c > 0 takes there: the sign of the scale is in Q, and a scale of 0 becomes
  // tiny so that the -inf of a dead key stays -inf
  uint32_t eight[4];  // A operand of the -8: rows 2 n, 2 n + 1 take group n
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    eight[n] = (r >> 1) == n ? 0x00080008u : 0u;
    asm("" : "+r"(eight[n]));
  }
  const float to_cap = a.scale * kTwo24 / a.softcap, cap_log2 = a.softcap * kLog2e;  // CAP only
  const float c_log2 = CAP ? 1.0f : fmaxf(fabsf(a.scale) * (kLog2e * kTwo24), 1e-30f), inv_c = 1.0f / c_log2;
  uint32_t slot = 0, refill = (kStages - kStep) * kSlot;  // byte offsets in the ring
  for (int k = 0; k < nt; k += kStep) {
    if ((k & 31) == 0 && k != 0) {
      sm_blk[warp][(k + kBlkRing - 64 + lane) & (kBlkRing - 1)] = ahead;
      ahead = block_number(k + kBlkRing - 32 + lane);
    }
    __syncwarp();  // also: the slots refilled here were read in the last step
    int blk[kStep];
#pragma unroll
    for (int u = 0; u < kStep; ++u) {
      blk[u] = sm_blk[warp][(k + u) & (kBlkRing - 1)];
      issue(sm_blk[warp][(k + u + kStages - kStep) & (kBlkRing - 1)], refill + u * kSlot);
    }
    copy_commit();
    copy_wait<kStages / kStep - 1>();
    __syncwarp();
    float x[kStep][4];
    uint4 vw[kStep][2], vs[kStep][2];
    uint32_t vmax = v_lim;  // scales are not negative, so they order as 16-bit integers
#pragma unroll
    for (int u = 0; u < kStep; ++u) {
      const uint32_t kb = wbase + slot + u * kSlot, vb = kb + kI4Block;
      uint4 kw[2];
      uint2 ks[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        kw[h] = lds128(kb + 512 * h + 16 * lane);     // token r + 8 h
        ks[h] = lds64(kb + kI4Codes + 64 * h + 8 * r);
        vw[u][h] = lds128(vb + 512 * h + 16 * lane);  // tokens 2 t, 2 t + 1 (+ 8 h)
        vs[u][h] = lds128(vb + kI4Codes + 64 * h + 16 * t);
      }
      // ---- S = K Q^T: rows token r / r + 8, columns heads 2 t, 2 t + 1 ---------
      float s[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const uint32_t w0 = word(kw[0], n), w1 = word(kw[1], n);
        const uint32_t y0 = w0 >> 8, y1 = w1 >> 8;
        float c[4];
        mma_from(c, w0 & kLo, w1 & kLo, y0 & kLo, y1 & kLo, qb[n][0], qb[n][2], qinit[n][0], qinit[n][1], qinit[n][2],
                 qinit[n][3]);
        mma_16816(c, w0 & kHi, w1 & kHi, y0 & kHi, y1 & kHi, qb[n][1], qb[n][3]);
        const float2 sa = f2(n < 2 ? ks[0].x : ks[0].y), sb = f2(n < 2 ? ks[1].x : ks[1].y);
        const float s0 = (n & 1) ? sa.y : sa.x, s1 = (n & 1) ? sb.y : sb.x;
        s[0] = n ? fmaf(s0, c[0], s[0]) : s0 * c[0];
        s[1] = n ? fmaf(s0, c[1], s[1]) : s0 * c[1];
        s[2] = n ? fmaf(s1, c[2], s[2]) : s1 * c[2];
        s[3] = n ? fmaf(s1, c[3], s[3]) : s1 * c[3];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) x[u][i] = CAP ? cap_log2 * tanhf(s[i] * to_cap) : s[i];
    }
    refill = slot;
    slot = slot == (kStages - kStep) * kSlot ? 0 : slot + kStep * kSlot;
    // dead keys: what stands there (codes, scales) may be anything
    if ((blk[0] | blk[kStep - 1]) < 0) {
#pragma unroll
      for (int u = 0; u < kStep; ++u) {
        const int pos0 = (first + kWarps * (k + u)) << 4;
        const int lo = min_key, hi = blk[u] == kDead ? 0 : seq_len;
        if (pos0 + r < lo || pos0 + r >= hi) x[u][0] = x[u][1] = -INFINITY;
        if (pos0 + r + 8 < lo || pos0 + r + 8 >= hi) x[u][2] = x[u][3] = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = pos0 + 2 * t + 8 * h;
          const uint32_t keep = (key >= lo && key < hi ? 0x0000ffffu : 0u) |
                                (key + 1 >= lo && key + 1 < hi ? 0xffff0000u : 0u);
          vs[u][h].x &= keep; vs[u][h].y &= keep; vs[u][h].z &= keep; vs[u][h].w &= keep;
        }
      }
    }

    // ---- the reference moves when a score or a V scale outgrows it -------------
    float mx[2] = {fmaxf(x[0][0], x[0][2]), fmaxf(x[0][1], x[0][3])};
#pragma unroll
    for (int u = 0; u < kStep; ++u) {
      if (u) {
        mx[0] = fmaxf(mx[0], fmaxf(x[u][0], x[u][2]));
        mx[1] = fmaxf(mx[1], fmaxf(x[u][1], x[u][3]));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
        vmax = __vimax3_u16x2(__vimax3_u16x2(vmax, vs[u][h].x, vs[u][h].y), vs[u][h].z, vs[u][h].w);
    }
    const bool grow = mx[0] > m_lim[0] || mx[1] > m_lim[1] || vmax != v_lim;
    if (__any_sync(0xffffffffu, grow)) {
      const float2 vf = f2(vmax);  // at least 2^v_exp
      const float vm = warp_max(fmaxf(vf.x, vf.y));
      int e = v_exp;
      if (vm > f2(v_lim).x) e = min(15, (int)((__float_as_uint(vm) >> 23) & 255) - 126);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], o));
        // reference = score maximum + exponent of the V scales - 4: p <= 2^15
        // and s p <= 2^12 while a score may still outgrow the maximum by 2^8
        const float base = m_ref[j] - (float)(v_exp - 4);
        const float top = fmaxf(base, mx[j] * c_log2), m_new = top + (float)(e - 4);
        const float corr = ex2(m_ref[j] - m_new);
        m_ref[j] = m_new;
        m_lim[j] = (top + 8.0f) * inv_c;
        l_run[j] *= corr;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc[i][j] *= corr;
          acc[i][2 + j] *= corr;
        }
        off[j] *= corr;
      }
      v_exp = e;
      v_lim = (uint32_t)(e + 15) * 0x04000400u;
    }

#pragma unroll
    for (int u = 0; u < kStep; ++u) {
      float p[4];
      p[0] = ex2(fmaf(x[u][0], c_log2, -m_ref[0]));
      p[1] = ex2(fmaf(x[u][1], c_log2, -m_ref[1]));
      p[2] = ex2(fmaf(x[u][2], c_log2, -m_ref[0]));
      p[3] = ex2(fmaf(x[u][3], c_log2, -m_ref[1]));
      l_run[0] += p[0] + p[2];
      l_run[1] += p[1] + p[3];
      const uint32_t p0 = transpose8x8(pack_half2(p[0], p[1]));  // head r, tokens 2 t, 2 t + 1
      const uint32_t p1 = transpose8x8(pack_half2(p[2], p[3]));  // tokens + 8

      // ---- O^T += V^T (s P)^T: m-block 2 n + j = dims 32 n + 4 row' + {2 j, 2 j + 1}
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const uint32_t b0 = hmul2(p0, word(vs[u][0], n)), b1 = hmul2(p1, word(vs[u][1], n));
        const uint32_t w0 = word(vw[u][0], n), w1 = word(vw[u][1], n);
        const uint32_t y0 = prmt(w0, 0u, 0x4341u), y1 = prmt(w1, 0u, 0x4341u);  // bytes 1 and 3
        mma_16816(acc[2 * n], w0 & kLo, w0 & kBoth, w1 & kLo, w1 & kBoth, b0, b1);
        mma_16816(acc[2 * n + 1], y0 & kLo, y0, y1 & kLo, y1, b0, b1);
        mma_16816(off, eight[n], 0u, eight[n], 0u, b0, b1);
      }
    }
  }

  // ---- join the warps of this split (O staged in this warp's own ring) ---------
  copy_wait<0>();
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) l_run[j] += __shfl_xor_sync(0xffffffffu, l_run[j], o);
    if (r == 0) {
      sm_m[warp][2 * t + j] = m_ref[j];
      sm_l[warp][2 * t + j] = l_run[j];
    }
  }
  float* my_o = reinterpret_cast<float*>(ring + warp * kWarpBytes);  // [8][128]
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float o8 = __shfl_sync(0xffffffffu, off[j], 8 * n + t);  // row 2 n
      const float lo0 = acc[2 * n][j], lo1 = acc[2 * n + 1][j];
      const float hi0 = (acc[2 * n][2 + j] - lo0) * 0.0625f, hi1 = (acc[2 * n + 1][2 + j] - lo1) * 0.0625f;
      const float4 v = make_float4((lo0 - o8) * kTwo24, (hi0 - o8) * kTwo24, (lo1 - o8) * kTwo24, (hi1 - o8) * kTwo24);
      *reinterpret_cast<float4*>(my_o + (2 * t + j) * kD + 32 * n + 4 * r) = v;
    }
  __syncthreads();

  const int dim = threadIdx.x;  // 128 threads == head dim
  const size_t out_row = ((size_t)b * a.num_heads + (size_t)g * group) * kD;
  auto store = [&](int h, int d, float o, float l) {
    const float v = l != 0.0f ? o / l : 0.0f;
    if (a.out_bf16)
      reinterpret_cast<__nv_bfloat16*>(a.out)[out_row + (size_t)h * kD + d] = __float2bfloat16_rn(v);
    else
      a.out[out_row + (size_t)h * kD + d] = v;
  };
  const bool whole = SHARES ? nparts == 1 : nparts == 0;
  // where this CTA's partial row goes
  const size_t slot_at = SHARES ? 2 * (size_t)blockIdx.x + (first_row ? 0 : 1) : row * a.max_parts + part;
  float* cta_o = reinterpret_cast<float*>(ring);  // [8][128], over the first warp's
  for (int h = 0; h < group; ++h) {
    float M = kNone, O = 0.0f, L = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w][h]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = ex2(sm_m[w][h] - M);
      O += f * reinterpret_cast<const float*>(ring + w * kWarpBytes)[h * kD + dim];
      L += f * sm_l[w][h];
    }
    if (whole) {
      store(h, dim, O, L);
    } else if (slices == 1) {
      a.part_o[(slot_at * group + h) * kD + dim] = O;
      if (dim == 0) {
        a.part_ml[(slot_at * group + h) * 2] = M;
        a.part_ml[(slot_at * group + h) * 2 + 1] = L;
      }
    } else {
      cta_o[h * kD + dim] = O;  // read only by this thread before
      if (dim == 0) {
        cta_ml[h][0] = M;
        cta_ml[h][1] = L;
      }
    }
  }
  if (whole) {
    if (SHARES) continue;
    return;
  }

  // ---- the splits of a cluster: this CTA joins its slice of the dims ------------
  int rank = 0;
  const int width = kD / slices;
  if (!SHARES && slices > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    rank = (int)cluster.block_rank();
    cluster.sync();
    for (int i = threadIdx.x; i < group * width; i += kWarps * 32) {
      const int h = i / width, d = rank * width + i % width;
      float M = kNone, O = 0.0f, L = 0.0f;
      float m[8], o[8], l[8];
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < slices) {
          const float* ml = cluster.map_shared_rank(&cta_ml[h][0], c);
          m[c] = ml[0];
          l[c] = ml[1];
          o[c] = cluster.map_shared_rank(cta_o, c)[h * kD + d];
          M = fmaxf(M, m[c]);
        }
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < slices) {
          const float f = ex2(m[c] - M);
          O += f * o[c];
          L += f * l[c];
        }
      if (nparts == 1) {
        store(h, d, O, L);
      } else {
        a.part_o[(slot_at * group + h) * kD + d] = O;
        if (i % width == 0) {
          float* ml = a.part_ml + ((slot_at * slices + rank) * group + h) * 2;
          ml[0] = M;
          ml[1] = L;
        }
      }
    }
    cluster.sync();  // the others have read this CTA's partials
    if (nparts == 1) return;
  }
  // ---- the last part of (b, g, slice) to finish stitches them, in order --------
  int c0 = 0;       // SHARES: the CTA that holds the row's first block,
  bool c0_second = false;  // as the second part that it writes
  if (SHARES) {
    const int size = sm_end[b] - (b ? sm_end[b - 1] : 0);
    c0 = share.owner(row_at);
    nparts = share.owner(row_at + size - 1) - c0 + 1;
    c0_second = share.begin(c0) < row_at;
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned* counter = &a.counters[row * slices + rank];
    sm_last = atomicAdd(counter, 1u) == (unsigned)(nparts - 1);
    if (sm_last) *counter = 0u;  // ready for the next launch
  }
  __syncthreads();
  if (sm_last) {
    __threadfence();
    for (int i = threadIdx.x; i < group * width; i += kWarps * 32) {
      const int h = i / width, d = rank * width + i % width;
      float M = kNone, O = 0.0f, L = 0.0f;
      // a running reference, so that the loads of several parts are in flight
      constexpr int kBatch = 8;
      for (int p0 = 0; p0 < nparts; p0 += kBatch) {
        float2 ml[kBatch];
        float o[kBatch];
#pragma unroll
        for (int c = 0; c < kBatch; ++c) {
          const int p = min(p0 + c, nparts - 1);
          const size_t from =
              SHARES ? 2 * (size_t)(c0 + p) + (p == 0 && c0_second ? 1 : 0) : row * a.max_parts + p;
          ml[c] = __ldcg(reinterpret_cast<const float2*>(a.part_ml) + (from * slices + rank) * group + h);
          o[c] = __ldcg(a.part_o + (from * group + h) * kD + d);
        }
        float m = M;
#pragma unroll
        for (int c = 0; c < kBatch; ++c) m = fmaxf(m, ml[c].x);
        const float f0 = ex2(M - m);
        O *= f0;
        L *= f0;
        M = m;
#pragma unroll
        for (int c = 0; c < kBatch; ++c)
          if (p0 + c < nparts) {
            const float f = ex2(ml[c].x - M);
            O += f * o[c];
            L += f * ml[c].y;
          }
      }
      store(h, d, O, L);
    }
  }
  if (!SHARES) return;
  }  // rows of the share
}

template <bool CAP, bool SHARES>
int launch_one(const Args& a, dim3 grid, unsigned slices, cudaStream_t st) {
  static std::atomic<bool> attr[kMaxDevices];
  const int rc = once_per_device(attr, [] {
    return cuda_status(
        cudaFuncSetAttribute(decode_kernel<CAP, SHARES>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem),
        "cudaFuncSetAttribute(paged_decode_int4)");
  });
  if (rc != DOE_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = slices;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = slices > 1 ? 2 : 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, decode_kernel<CAP, SHARES>, a), "paged_decode_int4");
}

// How a launch is cut, and the sizes that follow.
struct Plan {
  bool shares;                     // even shares of all rows' blocks over `grid` CTAs
  uint64_t split_tiles, slices;    // else: blocks per split, splits per cluster
  uint64_t max_parts, grid;        // parts per row, CTAs (per row when not shares)
  uint64_t slots;                  // partial rows in the workspace
};

// Even shares while a row is cut into a few parts at most, which its last CTA
// stitches alone.  With fewer rows than that each row gets its own splits, so
// many that there are about two CTAs per SM, joined in clusters.  A given
// split_pages asks for splits of that length; they serve more than
// kMaxStreamSeqs sequences too.
Plan plan(uint64_t num_seqs, uint64_t kv_heads, uint64_t max_tiles, uint64_t tiles_per_page, uint64_t split_pages) {
  Plan p = {};
  const uint64_t rows = num_seqs * kv_heads, ctas = (uint64_t)num_sms() * kCtasPerSm;
  p.slices = 1;
  if (split_pages == 0 && num_seqs <= kMaxStreamSeqs && rows * 16 >= ctas && rows * max_tiles <= 0x7fffffffull) {
    p.shares = true;
    p.grid = ctas * (getenv("I4M") ? atoi(getenv("I4M")) : 1);
    p.max_parts = 2;
    p.slots = 2 * p.grid;
    return p;
  }
  uint64_t t = split_pages * tiles_per_page;
  if (t == 0) {
    const uint64_t fill = (2 * (uint64_t)num_sms() + rows - 1) / rows;
    t = (max_tiles + fill - 1) / fill;
    if (t < 4) t = 4;
  }
  if (t > max_tiles) t = max_tiles;
  p.split_tiles = t;
  const uint64_t splits = (max_tiles + t - 1) / t;
  p.slices = splits > 16 ? 8 : 1;
  p.max_parts = (splits + p.slices - 1) / p.slices;
  p.grid = p.max_parts * p.slices;
  p.slots = rows * p.max_parts;
  return p;
}

}  // namespace i4

int launch_paged_decode_int4(const doe_paged_kv* kv, uint32_t num_seqs, uint32_t num_heads, const void* q,
                             const int32_t* seq_lens, const void* new_k, const void* new_v, float scale, float* out,
                             uint32_t split_pages, const doe_decode_options* opts, const doe_launch* launch,
                             uint64_t* ws_needed_out) {
  using namespace i4;
  const uint32_t Hkv = kv->num_kv_heads, group = num_heads / Hkv;
  const uint32_t tpp = kv->page_size / 16;
  const uint64_t max_tiles = (uint64_t)kv->max_pages_per_seq * tpp;
  const uint64_t rows = (uint64_t)num_seqs * Hkv;
  const Plan pl = plan(num_seqs ? num_seqs : 1, Hkv, max_tiles, tpp, split_pages);
  const uint64_t parts = pl.slots * group;
  const uint64_t ctr_off = (parts * (kD + 2 * pl.slices) * sizeof(float) + 255) / 256 * 256;
  const uint64_t ws = ctr_off + rows * pl.slices * sizeof(unsigned);
  if (ws_needed_out) {
    *ws_needed_out = ws;
    return DOE_OK;
  }
  if (group < 1 || group > 8) {
    set_op_error("doe_paged_decode: int4 pools take 1 to 8 heads per kv head (got %u)", group);
    return DOE_UNSUPPORTED;
  }
  if (launch->workspace == nullptr || launch->workspace_bytes < ws) {
    set_op_error("doe_paged_decode: workspace of %llu bytes required, %llu given", (unsigned long long)ws,
                 (unsigned long long)launch->workspace_bytes);
    return DOE_INVALID_ARGUMENT;
  }
  if (max_tiles * 16 > 0x7fffffffull || pl.grid > 0x7fffffffull || Hkv > 65535u ||
      (uint64_t)kv->num_pages * Hkv * tpp > 0x7fffffffull) {
    set_op_error("doe_paged_decode: more than 2^31 - 1 tokens in a block-table row or blocks in a pool, or over 65535 "
                 "kv heads");
    return DOE_INVALID_ARGUMENT;
  }
  for (const void* p : {(const void*)kv->k_pool, (const void*)kv->v_pool, q, (const void*)launch->workspace})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) {
      set_op_error("doe_paged_decode: pools, q and the workspace must be 16-byte aligned");
      return DOE_INVALID_ARGUMENT;
    }
  for (const void* p : {new_k, new_v})
    if (reinterpret_cast<uintptr_t>(p) % 8 != 0) {
      set_op_error("doe_paged_decode: new_k and new_v must be 8-byte aligned");
      return DOE_INVALID_ARGUMENT;
    }
  Args a;
  a.q = static_cast<const __half*>(q);
  a.k_pool = static_cast<uint8_t*>(kv->k_pool);
  a.v_pool = static_cast<uint8_t*>(kv->v_pool);
  a.block_table = kv->block_table;
  a.seq_lens = seq_lens;
  a.new_k = static_cast<const __half*>(new_k);
  a.new_v = static_cast<const __half*>(new_v);
  a.out = out;
  a.part_o = static_cast<float*>(launch->workspace);
  a.part_ml = a.part_o + parts * kD;
  a.counters = reinterpret_cast<unsigned*>(static_cast<uint8_t*>(launch->workspace) + ctr_off);
  a.status = launch->status;
  a.freq_cis = opts ? opts->freq_cis : nullptr;
  a.rope_positions = opts ? (int)opts->rope_positions : 0;
  a.window = opts ? (int)(opts->sliding_window > 0x7fffffffu ? 0x7fffffffu : opts->sliding_window) : 0;
  a.softcap = opts ? opts->attn_softcap : 0.0f;
  a.scale = scale;
  a.num_heads = (int)num_heads;
  a.num_kv_heads = (int)Hkv;
  a.group = (int)group;
  a.num_pages = (int)kv->num_pages;
  a.page_size = (int)kv->page_size;
  a.max_pages = (int)kv->max_pages_per_seq;
  a.tiles_per_page = (int)tpp;
  a.tile_shift = -1;
  for (int s = 0; s < 27; ++s)
    if (tpp == (1u << s)) a.tile_shift = s;
  a.num_seqs = (int)num_seqs;
  a.split_tiles = (int)pl.split_tiles;
  a.max_parts = (int)pl.max_parts;
  a.out_bf16 = (opts && (opts->flags & DOE_DECODE_OUT_BF16)) ? 1 : 0;
  a.inputs_stable = (opts && (opts->flags & DOE_DECODE_INPUTS_STABLE)) ? 1 : 0;
  cudaStream_t st = static_cast<cudaStream_t>(launch->stream);
  if (pl.max_parts > 1 && !(opts && (opts->flags & DOE_DECODE_COUNTERS_ZEROED))) {
    const int rc =
        cuda_status(cudaMemsetAsync(a.counters, 0, rows * pl.slices * sizeof(unsigned), st), "cudaMemsetAsync(split counters)");
    if (rc != DOE_OK) return rc;
  }
  const dim3 grid = pl.shares ? dim3((unsigned)pl.grid) : dim3((unsigned)pl.grid, Hkv, num_seqs);
  const unsigned slices = (unsigned)pl.slices;
  if (pl.shares)
    return a.softcap > 0.0f ? launch_one<true, true>(a, grid, slices, st) : launch_one<false, true>(a, grid, slices, st);
  return a.softcap > 0.0f ? launch_one<true, false>(a, grid, slices, st) : launch_one<false, false>(a, grid, slices, st);
}

}  // namespace doe
