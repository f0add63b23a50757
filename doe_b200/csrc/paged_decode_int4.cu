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
// Loads: one warp consumes one 16-token block per step out of a ring of its own
// that two bulk copies (K block, V block, 1152 contiguous bytes each) fill.
#include "int4.cuh"
#include "tma.cuh"

namespace doe {
namespace i4 {

constexpr int kD = 128;
constexpr int kWarps = 4;
constexpr int kStages = 4;
constexpr int kPageRegs = 4;                   // page ids per lane: 128 blocks per warp, 512 per split
constexpr int kMaxSplitTiles = kWarps * 32 * kPageRegs;
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
  float* part_o;        // [B * Hkv * max_splits, group, 128]
  float* part_ml;       // [B * Hkv * max_splits, group, 2]
  unsigned* counters;   // [B * Hkv], zero at launch, left zero by the stitch
  int32_t* status;
  const float* freq_cis;
  int rope_positions;
  int window;
  float softcap;
  float scale;
  int num_heads, num_kv_heads, group, num_pages, page_size, max_pages;
  int tiles_per_page, tile_shift;  // page_size / 16 and its log2 (-1: not a power of two)
  int split_tiles, max_splits;
  int out_bf16;
  int inputs_stable;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
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

  // Ends with the fence that lets this warp's later bulk copies read the row.
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
    asm volatile("fence.proxy.async.global;\n" ::: "memory");
    __syncwarp();
  }
};

constexpr uint32_t kLo = 0x000f000fu, kHi = 0x00f000f0u;
constexpr float kTwo24 = 16777216.0f;

template <bool CAP>
__global__ void __launch_bounds__(kWarps * 32) decode_kernel(const Args a) {
  extern __shared__ __align__(128) uint8_t ring[];
  if (!a.inputs_stable) pdl_wait();
  const int split = blockIdx.x, g = blockIdx.y, b = blockIdx.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, t = lane & 3;
  const int Hkv = a.num_kv_heads, group = a.group;

  const int raw_len = a.seq_lens[b];
  const int cap = a.max_pages * a.page_size;
  const int seq_len = raw_len < 0 ? 0 : (raw_len > cap ? cap : raw_len);
  if (raw_len != seq_len && split == 0 && g == 0 && threadIdx.x == 0) report(a.status, DOE_DEVICE_ERR_LENGTH);
  // window: keys [min_key, seq_len); the walk starts at the block holding min_key
  const int min_key = (a.window > 0 && seq_len > a.window) ? seq_len - a.window : 0;
  const int tile_origin = min_key >> 4;
  const int ntiles = ((seq_len + 15) >> 4) - tile_origin;
  const int nsplits = max(1, (ntiles + a.split_tiles - 1) / a.split_tiles);
  if (split >= nsplits) return;
  const int tile_begin = split * a.split_tiles;  // relative to tile_origin
  const int tile_end = min(ntiles, tile_begin + a.split_tiles);
  const int32_t* table = a.block_table + (size_t)b * a.max_pages;

  __shared__ float sm_m[kWarps][8];
  __shared__ float sm_l[kWarps][8];
  __shared__ int sm_last;
  __shared__ int sm_pg[kWarps][32 * kPageRegs];
  __shared__ __align__(8) uint64_t ring_bar[kWarps][kStages];

  if (lane == 0) {
#pragma unroll
    for (int st = 0; st < kStages; ++st) mbar_init(smem_addr(&ring_bar[warp][st]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncwarp();

  // this warp's blocks: first + kWarps * k, k < nt; page ids up front
  const int first = tile_origin + tile_begin + warp;
  const int span = tile_end - tile_begin - warp;
  const int nt = span > 0 ? (span + kWarps - 1) / kWarps : 0;
  auto page_index = [&](int tile) { return a.tile_shift >= 0 ? tile >> a.tile_shift : tile / a.tiles_per_page; };
#pragma unroll
  for (int i = 0; i < kPageRegs; ++i)
    if (lane + 32 * i < nt) sm_pg[warp][lane + 32 * i] = table[page_index(first + kWarps * (lane + 32 * i))];
  __syncwarp();

  const uint32_t wbase = smem_addr(ring) + warp * kWarpBytes;
  // Fills slot k % kStages with block k (whole warp calls, one lane issues).  A
  // block of a bad page gets a plain arrival; the consumer reports the page.
  auto issue = [&](int k) {
    if (lane != 0) return;
    const int page = sm_pg[warp][k];
    const uint32_t bar = smem_addr(&ring_bar[warp][k % kStages]);
    if ((unsigned)page >= (unsigned)a.num_pages) {
      mbar_arrive(bar);
      return;
    }
    const int tile = first + kWarps * k;
    const int in_page = tile - page_index(tile) * a.tiles_per_page;
    const size_t off = (((size_t)page * Hkv + g) * a.tiles_per_page + in_page) * kI4Block;
    const uint32_t dst = wbase + (k % kStages) * kSlot;
    // this warp read the slot's previous block through the generic proxy
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    mbar_expect_tx(bar, kSlot);
    bulk_load(dst, a.k_pool + off, kI4Block, bar);
    bulk_load(dst + kI4Block, a.v_pool + off, kI4Block, bar);
  };

  // first copies before the query work (and before griddepcontrol.wait when the
  // caller vouches for the inputs), except the block the append writes
  const bool appends = a.new_k != nullptr && split == nsplits - 1 && seq_len > 0;
  const int new_tile = ((seq_len - 1) >> 4) - tile_origin - tile_begin;  // split-relative
  int issued = 0;
  for (; issued < kStages - 1 && issued < nt; ++issued)
    if (appends && new_tile == warp + kWarps * issued) break;
    else issue(issued);
  if (a.inputs_stable) pdl_wait();
  pdl_trigger();

  // the warp whose walk holds the new row's block appends the row itself
  const bool append_pending = appends && new_tile % kWarps == warp;
  AppendRow app;
  if (append_pending) app.load(a, b, g, seq_len - 1, table, lane);

  // ---- Q as the B operand: lane (r = head, t) holds dims 32 grp + 8 t + 0..7,
  // word i of each run = dims (2 i, 2 i + 1) = the K word's nibbles i and i + 4
  uint32_t qb[4][4];
  float qinit[4][2];  // -8 sum_group q of heads 2 t, 2 t + 1 (times 2^-24)
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
                      split == 0 && g == 0 && lane == 0 && warp == 0, rc, rsn);
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
        uint32_t w = word(qv[n], i);
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
      for (int j = 0; j < 2; ++j) qinit[n][j] = -8.0f / kTwo24 * __shfl_sync(0xffffffffu, qs, (2 * t + j) * 4);
    }
  }

  // heads 2 t and 2 t + 1 of this lane's accumulator columns
  float m_ref[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.0f, 0.0f};
  int v_exp = -3;             // every V scale seen is below 2^v_exp (or at the clamp)
  uint32_t v_lim = 0x30003000u;  // 2^v_exp as an f16 pair
  float acc[8][4], off[4][4];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) off[i][0] = off[i][1] = off[i][2] = off[i][3] = 0.0f;

  if (append_pending) app.store(a, g, lane);
  for (int s0 = issued; s0 < kStages - 1; ++s0)
    if (s0 < nt) issue(s0);

  const float to_log2 = CAP ? a.scale * kTwo24 / a.softcap : a.scale * kLog2e * kTwo24;
  const float cap_log2 = CAP ? a.softcap * kLog2e : 0.0f;
  for (int k = 0; k < nt; ++k) {
    __syncwarp();
    if (k + kStages - 1 < nt) issue(k + kStages - 1);
    // block k has landed (bounded: a timeout ends this warp's walk)
    if (!__all_sync(0xffffffffu,
                    mbar_wait_bounded(smem_addr(&ring_bar[warp][k % kStages]), (k / kStages) & 1))) {
      if (lane == 0) report(a.status, DOE_DEVICE_ERR_TIMEOUT);
      // the ring is reused below: wait (bounded) for the copies in flight
      for (int i = k + 1; i < nt && i < k + kStages; ++i)
        mbar_wait_bounded(smem_addr(&ring_bar[warp][i % kStages]), (i / kStages) & 1);
      break;
    }
    if ((unsigned)sm_pg[warp][k] >= (unsigned)a.num_pages) {
      if (lane == 0) report(a.status, DOE_DEVICE_ERR_PAGE);
      continue;
    }
    const int pos0 = (first + kWarps * k) << 4;
    const uint32_t kb = wbase + (k % kStages) * kSlot, vb = kb + kI4Block;
    uint4 kw[2], vw[2], vs[2];
    uint2 ks[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      kw[h] = lds128(kb + 512 * h + 16 * lane);             // token r + 8 h
      ks[h] = lds64(kb + kI4Codes + 64 * h + 8 * r);
      vw[h] = lds128(vb + 512 * h + 16 * lane);             // tokens 2 t, 2 t + 1 (+ 8 h)
      vs[h] = lds128(vb + kI4Codes + 64 * h + 16 * t);
    }

    // ---- S = K Q^T: rows token r / r + 8, columns heads 2 t, 2 t + 1 -----------
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const uint32_t w0 = word(kw[0], n), w1 = word(kw[1], n);
      const uint32_t y0 = w0 >> 8, y1 = w1 >> 8;
      float c[4] = {qinit[n][0], qinit[n][1], qinit[n][0], qinit[n][1]};
      mma_16816(c, w0 & kLo, w1 & kLo, y0 & kLo, y1 & kLo, qb[n][0], qb[n][2]);
      mma_16816(c, w0 & kHi, w1 & kHi, y0 & kHi, y1 & kHi, qb[n][1], qb[n][3]);
      const float2 sa = f2(n < 2 ? ks[0].x : ks[0].y), sb = f2(n < 2 ? ks[1].x : ks[1].y);
      const float s0 = (n & 1) ? sa.y : sa.x, s1 = (n & 1) ? sb.y : sb.x;
      s[0] = fmaf(s0, c[0], s[0]);
      s[1] = fmaf(s0, c[1], s[1]);
      s[2] = fmaf(s1, c[2], s[2]);
      s[3] = fmaf(s1, c[3], s[3]);
    }
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = CAP ? cap_log2 * tanhf(s[i] * to_log2) : s[i] * to_log2;
    // only the window's first block and the sequence's last hold dead keys; what
    // stands there (codes, scales) may be anything
    if (pos0 < min_key || pos0 + 16 > seq_len) {
      const bool live0 = pos0 + r >= min_key && pos0 + r < seq_len;
      const bool live1 = pos0 + r + 8 >= min_key && pos0 + r + 8 < seq_len;
      if (!live0) x[0] = x[1] = -INFINITY;
      if (!live1) x[2] = x[3] = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = pos0 + 2 * t + 8 * h;
        const uint32_t keep = (key >= min_key && key < seq_len ? 0x0000ffffu : 0u) |
                              (key + 1 >= min_key && key + 1 < seq_len ? 0xffff0000u : 0u);
        vs[h].x &= keep; vs[h].y &= keep; vs[h].z &= keep; vs[h].w &= keep;
      }
    }

    // ---- the reference moves when a score or a V scale outgrows it -------------
    const uint32_t vmax = hmax2(hmax2(hmax2(vs[0].x, vs[0].y), hmax2(vs[0].z, vs[0].w)),
                                hmax2(hmax2(vs[1].x, vs[1].y), hmax2(vs[1].z, vs[1].w)));
    const bool grow = fmaxf(x[0], x[2]) > m_ref[0] + 8.0f || fmaxf(x[1], x[3]) > m_ref[1] + 8.0f ||
                      !__hble2(*reinterpret_cast<const __half2*>(&vmax), *reinterpret_cast<const __half2*>(&v_lim));
    if (__any_sync(0xffffffffu, grow)) {
      const float2 vf = f2(vmax);
      const float vm = warp_max(fmaxf(vf.x, vf.y));
      int e = v_exp;
      if (vm > 0.0f) e = max(e, min(15, (int)((__float_as_uint(vm) >> 23) & 255) - 126));
      float mx[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], o));
        // reference = score maximum + exponent of the V scales - 4: p <= 2^15
        // and s p <= 2^12 while a score may still outgrow the maximum by 2^8
        const float base = m_ref[j] - (float)(v_exp - 4);
        const float m_new = (mx[j] > base + 8.0f || base == -INFINITY ? mx[j] : base) + (float)(e - 4);
        const float corr = m_ref[j] == -INFINITY ? 0.0f : ex2(m_ref[j] - m_new);
        m_ref[j] = m_new;
        l_run[j] *= corr;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc[i][j] *= corr;
          acc[i][2 + j] *= corr;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) off[i][j] *= corr;
      }
      v_exp = e;
      v_lim = e >= 16 ? 0x7bff7bffu : (uint32_t)(e + 15) * 0x04000400u;
    }

    float p[4];
    p[0] = ex2(x[0] - m_ref[0]);
    p[1] = ex2(x[1] - m_ref[1]);
    p[2] = ex2(x[2] - m_ref[0]);
    p[3] = ex2(x[3] - m_ref[1]);
    l_run[0] += p[0] + p[2];
    l_run[1] += p[1] + p[3];
    const uint32_t p0 = transpose8x8(pack_half2(p[0], p[1]));  // head r, tokens 2 t, 2 t + 1
    const uint32_t p1 = transpose8x8(pack_half2(p[2], p[3]));  // tokens + 8

    // ---- O^T += V^T (s P)^T: m-block 2 n + j = dims 32 n + 4 row' + {2 j, 2 j + 1}
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const uint32_t b0 = hmul2(p0, word(vs[0], n)), b1 = hmul2(p1, word(vs[1], n));
      const uint32_t w0 = word(vw[0], n), w1 = word(vw[1], n);
      const uint32_t y0 = w0 >> 8, y1 = w1 >> 8;
      mma_16816(acc[2 * n], w0 & kLo, w0 & kHi, w1 & kLo, w1 & kHi, b0, b1);
      mma_16816(acc[2 * n + 1], y0 & kLo, y0 & kHi, y1 & kLo, y1 & kHi, b0, b1);
      mma_16816(off[n], 0x00080008u, 0x00080008u, 0x00080008u, 0x00080008u, b0, b1);
    }
  }

  // ---- merge the warps of this split (O staged in this warp's own ring) --------
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
  __syncwarp();
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float o8 = off[n][j];
      const float4 v = make_float4((acc[2 * n][j] - o8) * kTwo24, (acc[2 * n][2 + j] * 0.0625f - o8) * kTwo24,
                                   (acc[2 * n + 1][j] - o8) * kTwo24, (acc[2 * n + 1][2 + j] * 0.0625f - o8) * kTwo24);
      *reinterpret_cast<float4*>(my_o + (2 * t + j) * kD + 32 * n + 4 * r) = v;
    }
  __syncthreads();

  const int dim = threadIdx.x;  // 128 threads == head dim
  const size_t out_row = ((size_t)b * a.num_heads + (size_t)g * group) * kD;
  auto store = [&](int h, float v) {
    if (a.out_bf16)
      reinterpret_cast<__nv_bfloat16*>(a.out)[out_row + (size_t)h * kD + dim] = __float2bfloat16_rn(v);
    else
      a.out[out_row + (size_t)h * kD + dim] = v;
  };
  const size_t base = ((size_t)b * Hkv + g) * a.max_splits;
  for (int h = 0; h < group; ++h) {
    float M = -INFINITY, O = 0.0f, L = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm_m[w][h]);
    if (M != -INFINITY) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2f(sm_m[w][h] - M);  // -inf -> 0
        O += f * reinterpret_cast<const float*>(ring + w * kWarpBytes)[h * kD + dim];
        L += f * sm_l[w][h];
      }
    }
    if (nsplits == 1) {
      store(h, L != 0.0f ? O / L : 0.0f);
    } else {
      const size_t prow = (base + split) * group + h;
      a.part_o[prow * kD + dim] = O;
      if (dim == 0) {
        a.part_ml[prow * 2] = M;
        a.part_ml[prow * 2 + 1] = L;
      }
    }
  }
  if (nsplits == 1) return;
  // ---- the last split of (b, g) to finish stitches them, in split order --------
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const unsigned old = atomicAdd(&a.counters[(size_t)b * Hkv + g], 1u);
    sm_last = old == (unsigned)(nsplits - 1);
    if (sm_last) a.counters[(size_t)b * Hkv + g] = 0u;  // ready for the next launch
  }
  __syncthreads();
  if (!sm_last) return;
  __threadfence();
  for (int h = 0; h < group; ++h) {
    float M = -INFINITY, O = 0.0f, L = 0.0f;
    for (int sp = 0; sp < nsplits; ++sp) M = fmaxf(M, __ldcg(a.part_ml + ((base + sp) * group + h) * 2));
    if (M != -INFINITY) {
      for (int sp = 0; sp < nsplits; ++sp) {
        const size_t prow = (base + sp) * group + h;
        const float f = exp2f(__ldcg(a.part_ml + prow * 2) - M);
        O += f * __ldcg(a.part_o + prow * kD + dim);
        L += f * __ldcg(a.part_ml + prow * 2 + 1);
      }
    }
    store(h, L != 0.0f ? O / L : 0.0f);
  }
}

template <bool CAP>
int launch_cap(const Args& a, dim3 grid, cudaStream_t st) {
  static std::atomic<bool> attr[kMaxDevices];
  const int rc = once_per_device(attr, [] {
    return cuda_status(
        cudaFuncSetAttribute(decode_kernel<CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem),
        "cudaFuncSetAttribute(paged_decode_int4)");
  });
  if (rc != DOE_OK) return rc;
  return cuda_status(launch_pdl(decode_kernel<CAP>, grid, dim3(kWarps * 32), kSmem, st, a), "paged_decode_int4");
}

// Blocks per split.  Long splits amortise a CTA's pipeline fill and stitch;
// where the (sequence, kv head) rows are few the length is cut until there are
// about two CTAs per SM.
uint32_t auto_split_tiles(uint64_t rows, uint64_t max_tiles) {
  const uint64_t want = (max_tiles * rows + 1775) / 1776;
  if (want >= 128) return 128;
  uint64_t s = (max_tiles + 127) / 128;
  const uint64_t fill = (280 + rows - 1) / rows;
  if (s < fill) s = fill;
  const uint64_t t = (max_tiles + s - 1) / s;
  return (uint32_t)(t < 4 ? 4 : t);
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
  uint64_t split_tiles = split_pages ? (uint64_t)split_pages * tpp : auto_split_tiles(rows ? rows : 1, max_tiles);
  if (split_tiles > kMaxSplitTiles) split_tiles = kMaxSplitTiles;  // prefetched page ids
  const uint64_t max_splits = (max_tiles + split_tiles - 1) / split_tiles;
  const uint64_t parts = rows * max_splits * group;
  const uint64_t ctr_off = (parts * (kD + 2) * sizeof(float) + 255) / 256 * 256;
  const uint64_t ws = ctr_off + rows * sizeof(unsigned);
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
  if (max_tiles * 16 > 0x7fffffffull || max_splits > 0x7fffffffull || Hkv > 65535u) {
    set_op_error("doe_paged_decode: a block-table row spans more than 2^31 - 1 tokens, or over 65535 kv heads");
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
  a.split_tiles = (int)split_tiles;
  a.max_splits = (int)max_splits;
  a.out_bf16 = (opts && (opts->flags & DOE_DECODE_OUT_BF16)) ? 1 : 0;
  a.inputs_stable = (opts && (opts->flags & DOE_DECODE_INPUTS_STABLE)) ? 1 : 0;
  cudaStream_t st = static_cast<cudaStream_t>(launch->stream);
  if (max_splits > 1 && !(opts && (opts->flags & DOE_DECODE_COUNTERS_ZEROED))) {
    const int rc =
        cuda_status(cudaMemsetAsync(a.counters, 0, rows * sizeof(unsigned), st), "cudaMemsetAsync(split counters)");
    if (rc != DOE_OK) return rc;
  }
  const dim3 grid((unsigned)max_splits, Hkv, num_seqs);
  return a.softcap > 0.0f ? launch_cap<true>(a, grid, st) : launch_cap<false>(a, grid, st);
}

}  // namespace doe
