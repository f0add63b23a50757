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
// core.  K's pair at bits 4-7 is left there and reads n * 2^-20, so 8 codes cost
// one shift and 4 ANDs.  A V byte is used whole as the row of its high nibble,
// (lo + 16 hi) * 2^-24, and the low nibble's sum comes off at the end: 8 codes
// cost 4 operations.  The powers of two go into Q (words of the high nibbles
// times 2^-4), the score scale (2^24) and the final accumulators; -8 becomes the
// S accumulators' start value (-8 sum q) and, for O, one MMA per group with a
// constant A operand (8) on the same B operand, so exactly the f16 (s p) that the
// product used is taken off.  P moves from the S accumulators (token rows) into
// the B operand (head columns) by movmatrix.  S, the softmax statistics and O are
// f32; P and s p are rounded to f16 (2^-11 relative at most, the f16 and int8
// kernels' choice).
//
// The running reference of a head, m, is its score maximum plus the exponent e of
// the largest V scale seen, where that is within [-3, 1]; larger and smaller scales are
// first multiplied by the power of two that takes e there, which comes off at the end.
// So p and s p stay within f16's range, and a key down to 2^-17 of the largest one's
// weight out of its subnormals, whatever the magnitude of V (scales below 2^-18 lose
// that range by as much).  The reference is lazy: it moves only when a score exceeds it
// by 2^8 or a V scale exceeds the exponent.
//
// Loads: a warp walks its blocks kStep at a time out of a ring of its own in
// shared memory, filled with cp.async: a block is 1024 + 128 contiguous bytes
// of K and of V, 5 instructions for the warp.  (One elected lane issuing two
// bulk copies costs the warp some 45 instructions, waits included, of 320 a
// block: 128 us for 64 sequences of 1k-8k tokens against 98.)
//
// Work, see plan().  Many long rows (sequence, kv head): the blocks of all
// sequences are one list cut into even pieces, each for one warp per kv head, so
// that ragged lengths leave no tail; a row that pieces' ends cut is stitched by the
// last of its warps to arrive.  Few rows: each is cut into splits, one CTA each,
// as many as its share of all blocks; with very few, 8 of them form a cluster and
// join in distributed shared memory, each CTA a slice of the dims, and the clusters
// are stitched per slice by the last one to arrive.  Short rows, many of them: one
// CTA each.  Pieces and splits follow from the lengths alone and sums go in the
// order of the keys, so results do not depend on timing.
//
// What bounds it (8 kv heads, 4 query heads each, f32 output): 64 sequences of 1k-8k
// tokens take 76.8 us for 341 MB (4.4 TB/s, 0.68 of the measured copy rate), 32 of
// 8k-32k 145 us for 756 MB (5.2 TB/s, 0.80); the same walk without its arithmetic
// 63 and 122 us.  Over the batch sizes that is a line, 0.38 ns a block (6.1 TB/s) and
// 20 us for a launch: its start (5 us until the first blocks arrive), the warps' uneven
// ends (14 us from the first third of them to the last, which weighting their pieces
// does not shorten) and the last stitch (8).  A block costs a warp about 225
// instructions (110 ALU, 65 FMA, 20 MMA), half of the issue slots.  One sequence of
// 130001 tokens (2 kv heads, 37.5 MB) takes 20 us: a launch, three dependent loads,
// 11 blocks a warp, and two joins of 3 us each.
#include <algorithm>
#include <cmath>

#include <cooperative_groups.h>

#include "int4.cuh"

namespace doe {
namespace i4 {

namespace cg = cooperative_groups;

constexpr int kD = 128;
constexpr int kWarps = 4;
constexpr int kStep = 2;                       // blocks per loop step
constexpr int kStages = 6;                     // ring slots, a multiple of kStep
constexpr int kBlkRing = 128;                  // block numbers per warp, renewed 32 at a time
constexpr int kCtasPerSm = 3;                  // resident: 168 registers a thread
constexpr int kRowCost = 4;                    // a sequence's fixed cost in the list, in blocks
constexpr int kMinPiece = 8;                   // entries; more than kRowCost, so that no piece is empty
constexpr uint64_t kListRows = 7;              // the list serves more rows than a 7th of the resident warps
constexpr uint64_t kShortRow = 128;            // blocks that one CTA walks alone when there are rows enough
constexpr uint64_t kLoneRow = 32;              // the same, when there are few rows (400 tokens: 6.4 us; in splits 7.5)
constexpr uint64_t kMinSplit = 16;             // blocks (8: 10.4 us for 1 x 4000 tokens, 16: 9.1; 1 x 1024 7.3, 7.8)
constexpr uint64_t kCounterBytes = 1 << 16;    // of the workspace's head, for 2048 rows' counters
constexpr uint32_t kMaxListSeqs = 1024;        // sequences whose lengths a CTA adds up
constexpr int kSlot = 2 * kI4Block;            // K block, V block
constexpr int kWarpBytes = kStages * kSlot;    // also holds the warp's O, 8 x 128 f32
constexpr int kSmem = kWarps * kWarpBytes;
static_assert(kWarpBytes >= 8 * kD * 4, "the join stages a warp's O in its ring");

struct Args {
  const __half* q;  // [B, H, 128]
  uint8_t* k_pool;  // blocks [num_pages, Hkv, page_size / 16]
  uint8_t* v_pool;
  const int32_t* block_table;
  const int32_t* seq_lens;
  const __half* new_k;  // [B, Hkv, 128] or null
  const __half* new_v;
  float* out;           // [B, H, 128] f32, or bf16 storage when out_bf16
  float* part_o;        // splits: [B * Hkv * max_parts, group, 128]; pieces: [pieces, 2, group, 128]
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
  int units;                   // or, when not 0: clusters per kv head, shared out by the lengths
  int out_bf16;
  int inputs_stable;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// tanh within 2^-20 of its size: its Taylor series to y^7 (the next term is 3e-7 of it at 1/4)
// and, from 1/4 on, 1 - 2 / (1 + e^2y), which cancels for small y.
__device__ __forceinline__ float tanh_of(float y) {
  const float t = y * y;
  const float series = y * fmaf(t, fmaf(t, fmaf(t, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
  const float closed = fmaf(-2.0f, rcp(1.0f + ex2(y * (2.0f * kLog2e))), 1.0f);
  return fabsf(y) < 0.25f ? series : closed;
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// A block's 16-byte copies of one lane (two of K codes, two of V codes, one of
// scales where `scales`), or none of them.
__device__ __forceinline__ void copy_block(uint32_t dst, const void* k, const void* v, uint32_t s_dst, const void* s,
                                           bool some, bool scales) {
  asm volatile(
      "{\n.reg .pred p, q;\n"
      "setp.ne.s32 p, %5, 0;\n"
      "setp.ne.and.s32 q, %6, 0, p;\n"
      "@p cp.async.cg.shared.global [%0], [%1], 16;\n"
      "@p cp.async.cg.shared.global [%0 + 512], [%1 + 512], 16;\n"
      "@p cp.async.cg.shared.global [%0 + 1152], [%2], 16;\n"
      "@p cp.async.cg.shared.global [%0 + 1664], [%2 + 512], 16;\n"
      "@q cp.async.cg.shared.global [%3], [%4], 16;\n}\n" ::"r"(dst),
      "l"(k), "l"(v), "r"(s_dst), "l"(s), "r"((int)some), "r"((int)scales)
      : "memory");
}
static_assert(kI4Block == 1152 && kI4Codes == 1024, "copy_block's offsets");
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
      float amax = max_nan(max_nan(fabsf(x01.x), fabsf(x01.y)), max_nan(fabsf(x23.x), fabsf(x23.y)));
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const __half sh = __float2half_rn(div7(amax));
      const float s = __half2float(sh);
      const float rs = inverse_of(s);
      const uint2 c01 = quantize_u4x2(x01, s, rs), c23 = quantize_u4x2(x23, s, rs);
      uint8_t* dst = (kv ? a.v_pool : a.k_pool) + block;
      if (kv == 0) {
        // even lanes hold dims 0..3 of the word's 8, odd lanes dims 4..7
        uint32_t w = ((c01.x & 15u) | (c01.y & 15u) << 16 | (c23.x & 15u) << 4 | (c23.y & 15u) << 20) << (8 * (lane & 1));
        w |= __shfl_xor_sync(0xffffffffu, w, 1);
        if ((lane & 1) == 0) *reinterpret_cast<uint32_t*>(dst + tok * 64 + ((lane & 7) >> 1) * 16 + group * 4) = w;
        if ((lane & 7) == 0) *reinterpret_cast<__half*>(dst + kI4Codes + (tok * 4 + group) * 2) = sh;
      } else {
        const uint32_t w = pack_u4x4(c01.x, c01.y, c23.x, c23.y);
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

constexpr int kDead = -1;        // no block number
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

// One warp's stretch of a row's blocks: first + STRIDE * k, k < nt.
struct Stretch {
  int b, g, seq_len, min_key;
  int first, nt;
  int row_at;  // pieces: where the row begins in the list
  bool whole;  // nobody else holds a part of the row
};

// What a warp keeps of a stretch: heads 2 t and 2 t + 1 are the lane's columns.
struct Sums {
  float m[2], l[2];   // reference and sum of p (of this lane's tokens)
  float acc[8][4];    // O^T: m-block 2 n + j, rows (lo, lo + 16 hi) of dims 32 n + 4 r + 2 j + {0, 1}
  float off[4];       // rows 2 n: 8 sum s p of group n
  float unit;         // of acc and off
};

// A warp's ring of blocks and the walk over a stretch.
template <bool CAP, int STRIDE>
struct Walker {
  const Args& a;
  int* numbers;     // [kBlkRing] block numbers
  uint32_t wbase;   // the ring
  int lane, r, t;
  int ahead = kDead;

  // The ring's first copies of a stretch go into the slots after the first
  // step's: those may still stage the last stretch's O.
  static constexpr uint32_t kSlot0 = kStep * kSlot;

  const uint8_t *k_lane, *v_lane, *s_lane;  // this lane's part of block 0
  uint32_t lane_dst, s_dst;
  bool bad = false;  // the stretch has blocks on bad pages

  __device__ __forceinline__ Walker(const Args& args, int* blk, void* ring, int l)
      : a(args), numbers(blk), wbase(smem_addr(ring)), lane(l), r(l >> 2), t(l & 3) {
    k_lane = a.k_pool + 16 * lane;
    v_lane = a.v_pool + 16 * lane;
    s_lane = (lane < 8 ? k_lane : v_lane - 128) + kI4Codes;
    lane_dst = wbase + 16 * lane;
    s_dst = lane_dst + kI4Codes + (lane < 8 ? 0 : kI4Block - 128);
  }

  // Page of the stretch's block i, and the block's number in the pools.  kDead:
  // past the walk, or on a page outside the pool.
  __device__ __forceinline__ int page_index(const Stretch& w, int i) const {
    const int tile = w.first + STRIDE * i;
    return a.tile_shift >= 0 ? tile >> a.tile_shift : tile / a.tiles_per_page;
  }
  __device__ __forceinline__ int page_of(const Stretch& w, int i) const {
    return i < w.nt ? a.block_table[(size_t)w.b * a.max_pages + page_index(w, i)] : kDead;
  }
  __device__ __forceinline__ int number_of(const Stretch& w, int i, int page) const {
    if (i >= w.nt) return kDead;
    const int tile = w.first + STRIDE * i;
    if ((unsigned)page < (unsigned)a.num_pages)
      return (page * a.num_kv_heads + w.g) * a.tiles_per_page + (tile - page_index(w, i) * a.tiles_per_page);
    report(a.status, DOE_DEVICE_ERR_PAGE);
    return kDead;
  }

  // Fills the slot at byte `slot` of the ring with block number blk, if it has one.
  // Lanes 0-7 copy the K scales, 8-15 the V scales.
  __device__ __forceinline__ void issue(int blk, uint32_t slot) const {
    const size_t off = (size_t)(uint32_t)blk * kI4Block;
    copy_block(lane_dst + slot, k_lane + off, v_lane + off, s_dst + slot, s_lane + off, blk >= 0, lane < 16);
  }

  // The block that receives the new row is the last of the warp that appends it.
  __device__ __forceinline__ bool appends(const Stretch& w) const {
    return a.new_k != nullptr && w.seq_len > 0 && w.nt > 0 && w.first + STRIDE * (w.nt - 1) == (w.seq_len - 1) >> 4;
  }
  // Blocks copied by start(): up to the ring's prefetch, not the one to be appended to.
  __device__ __forceinline__ int early(const Stretch& w) const {
    return min(kStages - kStep, appends(w) ? w.nt - 1 : w.nt);
  }

  // Looks the stretch's first block numbers up (96 ahead of the walk) and issues
  // its first copies.  Nothing of this warp is in flight.
  __device__ __forceinline__ void start(const Stretch& w) {
    int page[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) page[i] = page_of(w, 32 * i + lane);
#pragma unroll
    for (int i = 0; i < 3; ++i) numbers[32 * i + lane] = number_of(w, 32 * i + lane, page[i]);
    ahead = number_of(w, 96 + lane, page[3]);
    bool wrong = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) wrong |= 32 * i + lane < w.nt && (unsigned)page[i] >= (unsigned)a.num_pages;
    bad = __any_sync(0xffffffffu, wrong);
    static_assert(kBlkRing == 128, "three quarters are looked up, the fourth is ahead");
    __syncwarp();
    const int n = early(w);
    for (int k = 0; k < n; ++k) {
      issue(numbers[k], kSlot0 + k * kSlot);
      if (k % kStep == kStep - 1) copy_commit();
    }
  }

  // The rest: query, append, every block.  Leaves nothing in flight.
  __device__ __forceinline__ void walk(const Stretch& cur, Sums& sums) {
    const int g = cur.g, seq_len = cur.seq_len, min_key = cur.min_key, nt = cur.nt, first = cur.first;
    const int group = a.group;
    const bool append_pending = appends(cur);
    AppendRow app;
    if (append_pending) app.load(a, cur.b, g, seq_len - 1, a.block_table + (size_t)cur.b * a.max_pages, lane);

    // ---- Q as the B operand: lane (r = head, t) holds dims 32 grp + 8 t + 0..7,
    // word i of each run = dims (2 i, 2 i + 1) = the K word's nibbles i and i + 4
    uint32_t qb[4][4];
    float qinit[4][4];  // -8 sum_group q of heads 2 t, 2 t + 1 (times 2^-24), for both token rows
    {
      const __half* qrow = a.q + ((size_t)cur.b * a.num_heads + (size_t)g * group + r) * kD;
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
                        g == 0 && lane == 0, rc, rsn);
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

    float (&m_ref)[2] = sums.m;
    float (&l_run)[2] = sums.l;
    float (&acc)[8][4] = sums.acc;
    float (&off)[4] = sums.off;
    m_ref[0] = m_ref[1] = kNone;
    l_run[0] = l_run[1] = 0.0f;
    int v_exp = -18;               // every V scale seen is at most 2^v_exp (or infinite)
    uint32_t v_lim = 0x00400040u;  // 2^v_exp as an f16 pair
    uint32_t lift = 0x78007800u;   // 2^(middle(v_exp) - v_exp), what V scales are multiplied by, likewise
    auto middle = [](int e) { return min(max(e, -3), 1); };
    float m_lim[2] = {kNone, kNone};  // x of a score 2^8 over its maximum
    off[0] = off[1] = off[2] = off[3] = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;

    if (append_pending) app.store(a, g, lane);
    for (int k = early(cur); k < kStages - kStep; ++k) {
      issue(numbers[k], kSlot0 + k * kSlot);
      if (k % kStep == kStep - 1) copy_commit();
    }

    uint32_t eight[4];  // A operand of the -8: rows 2 n, 2 n + 1 take group n
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      eight[n] = (r >> 1) == n ? 0x00080008u : 0u;
      asm("" : "+r"(eight[n]));
    }
    // x is the softcapped score in the log2 domain (CAP) or the bare product, which
    // c > 0 takes there: the sign of the scale is in Q, and a scale of 0 becomes
    // tiny so that the -inf of a dead key stays -inf
    const float to_cap = fminf(fmaxf(kTwo24 * a.scale / a.softcap, -3e38f), 3e38f), cap_log2 = a.softcap * kLog2e;
    const float c_log2 = CAP ? 1.0f : fmaxf(fabsf(a.scale) * (kLog2e * kTwo24), 1e-30f), inv_c = 1.0f / c_log2;
    int edge_k = first * 16 < min_key || bad ? 0 : nt - kStep;  // steps from here on have dead keys
    uint32_t slot = kSlot0, refill = 0;  // byte offsets in the ring
    for (int k = 0; k < nt; k += kStep) {
      if ((k & 31) == 0 && k != 0) {
        numbers[(k + kBlkRing - 64 + lane) & (kBlkRing - 1)] = ahead;
        {
          const int i = k + kBlkRing - 32 + lane;
          ahead = number_of(cur, i, page_of(cur, i));
          bad |= __any_sync(0xffffffffu, i < nt && ahead == kDead);
        }
        // the -8 comes off the sums now and then: the tensor core truncates what it adds
        // to, and sums of codes from 1 on grow as sums of values do not (0.0020 of
        // O at 20000 tokens without this, 0.0004 with it)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float o8 = __shfl_sync(0xffffffffu, off[j], 8 * n + t);  // row 2 n
            acc[2 * n][j] -= o8;
            acc[2 * n + 1][j] -= o8;
            acc[2 * n][2 + j] = fmaf(-17.0f, o8, acc[2 * n][2 + j]);
            acc[2 * n + 1][2 + j] = fmaf(-17.0f, o8, acc[2 * n + 1][2 + j]);
          }
        off[0] = off[1] = off[2] = off[3] = 0.0f;
      }
      __syncwarp();  // also: the slots refilled here were read in the last step
      {
        const int2 blk = *reinterpret_cast<const int2*>(&numbers[(k + kStages - kStep) & (kBlkRing - 1)]);
        static_assert(kStep == 2, "block numbers are read in pairs");
        issue(blk.x, refill);
        issue(blk.y, refill + kSlot);
      }
      copy_commit();
      copy_wait<kStages / kStep - 1>();
      __syncwarp();
      float x[kStep][4];
      uint4 vs[kStep][2];
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
        for (int i = 0; i < 4; ++i)
          x[u][i] = CAP ? cap_log2 * tanh_of(s[i] * to_cap) : s[i];
      }
      const uint32_t v_at = wbase + slot + kI4Block + 16 * lane;
      refill = slot;
      slot = slot == (kStages - kStep) * kSlot ? 0 : slot + kStep * kSlot;
      // dead keys: in the window's first block, the sequence's last, blocks past the
      // walk and on bad pages; what stands there (codes, scales) may be anything
      const bool edge = k >= edge_k;
      edge_k = bad ? 0 : nt - kStep;
      if (edge) {
#pragma unroll
        for (int u = 0; u < kStep; ++u) {
          const int pos0 = (first + STRIDE * (k + u)) << 4;
          const int lo = min_key, hi = k + u >= nt || (bad && numbers[(k + u) & (kBlkRing - 1)] < 0) ? 0 : seq_len;
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
        const int mid = middle(e), drop = (mid - e) - (middle(v_exp) - v_exp);  // of the lift's exponent
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], o));
          // reference = score maximum + exponent of the lifted V scales - 4: p <= 2^15
          // and s p <= 2^12 while a score may still outgrow the maximum by 2^8
          const float base = m_ref[j] - (float)(middle(v_exp) - 4);
          const float top = fmaxf(base, mx[j] * c_log2), m_new = top + (float)(mid - 4);
          float corr = ex2(m_ref[j] - m_new);
          m_ref[j] = m_new;
          m_lim[j] = (top + 8.0f) * inv_c;
          l_run[j] *= corr;
          corr *= __uint_as_float((uint32_t)(127 + drop) << 23);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            acc[i][j] *= corr;
            acc[i][2 + j] *= corr;
          }
          off[j] *= corr;
        }
        v_exp = e;
        v_lim = e >= -14 ? (uint32_t)(e + 15) * 0x04000400u : 0x00010001u << (e + 24);
        lift = (uint32_t)(mid - e + 15) * 0x04000400u;
      }
      if (lift != 0x3c003c00u) {
#pragma unroll
        for (int u = 0; u < kStep; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            vs[u][h].x = hmul2(vs[u][h].x, lift);
            vs[u][h].y = hmul2(vs[u][h].y, lift);
            vs[u][h].z = hmul2(vs[u][h].z, lift);
            vs[u][h].w = hmul2(vs[u][h].w, lift);
          }
      }

#pragma unroll
      for (int u = 0; u < kStep; ++u) {
        const uint4 vw[2] = {lds128(v_at + u * kSlot), lds128(v_at + u * kSlot + 512)};  // tokens 2 t, 2 t + 1 (+ 8)
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
          const uint32_t w0 = word(vw[0], n), w1 = word(vw[1], n);
          const uint32_t y0 = prmt(w0, 0u, 0x4341u), y1 = prmt(w1, 0u, 0x4341u);  // bytes 1 and 3
          mma_16816(acc[2 * n], w0 & kLo, w0 & kBoth, w1 & kLo, w1 & kBoth, b0, b1);
          mma_16816(acc[2 * n + 1], y0 & kLo, y0, y1 & kLo, y1, b0, b1);
          mma_16816(off, eight[n], 0u, eight[n], 0u, b0, b1);
        }
      }
    }
    copy_wait<0>();
    __syncwarp();
    sums.unit = kTwo24 * __uint_as_float((uint32_t)(127 + v_exp - middle(v_exp)) << 23);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l_run[j] += __shfl_xor_sync(0xffffffffu, l_run[j], o);
  }

  // Calls put(column j, dim, four values) for the lane's share of O (not yet
  // divided by l): head 2 t + j, dims dim .. dim + 3.
  template <typename F>
  __device__ __forceinline__ void each(const Sums& s, F&& put) const {
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float o8 = __shfl_sync(0xffffffffu, s.off[j], 8 * n + t);  // row 2 n
        const float lo0 = s.acc[2 * n][j], lo1 = s.acc[2 * n + 1][j];
        const float hi0 = (s.acc[2 * n][2 + j] - lo0) * 0.0625f, hi1 = (s.acc[2 * n + 1][2 + j] - lo1) * 0.0625f;
        put(j, 32 * n + 4 * r,
            make_float4((lo0 - o8) * s.unit, (hi0 - o8) * s.unit, (lo1 - o8) * s.unit, (hi1 - o8) * s.unit));
      }
  }
};

// Output row (sequence, head), dims d .. d + 3: o / l, or 0 without keys.
__device__ __forceinline__ void store_out(const Args& a, size_t row, int d, float4 o, float l) {
  const float i = l != 0.0f ? 1.0f / l : 0.0f;
  const float4 v = make_float4(o.x * i, o.y * i, o.z * i, o.w * i);
  if (a.out_bf16) {
    const __nv_bfloat162 p[2] = {__floats2bfloat162_rn(v.x, v.y), __floats2bfloat162_rn(v.z, v.w)};
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(a.out) + row * kD + d) =
        *reinterpret_cast<const uint2*>(p);
  } else {
    *reinterpret_cast<float4*>(a.out + row * kD + d) = v;
  }
}

// Counts one part of a row in; true for the last of n.  The caller's threads have
// met at a barrier after their writes and meet at one before they read the parts.
__device__ __forceinline__ bool arrive_last(unsigned* counter, int n) {
  unsigned old;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;\n" : "=r"(old) : "l"(counter) : "memory");
  const bool last = old == (unsigned)(n - 1);
  if (last) *counter = 0u;  // ready for the next launch
  return last;
}

// A running sum of parts (m, l, o): eight are loaded together, then added in order.
struct Joined {
  static constexpr int kBatch = 8;
  float m = kNone, l = 0.0f;
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  // at(p, m l, o): the loads of part p < n
  template <typename F>
  __device__ __forceinline__ void add(int n, F&& at) {
    for (int p0 = 0; p0 < n; p0 += kBatch) {
      float2 ml[kBatch];
      float4 po[kBatch];
#pragma unroll
      for (int c = 0; c < kBatch; ++c) at(min(p0 + c, n - 1), ml[c], po[c]);
      float top = m;
#pragma unroll
      for (int c = 0; c < kBatch; ++c) top = fmaxf(top, ml[c].x);
      float f = ex2(m - top);
      o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
      l *= f;
      m = top;
#pragma unroll
      for (int c = 0; c < kBatch; ++c)
        if (p0 + c < n) {
          f = ex2(ml[c].x - m);
          o = make_float4(o.x + f * po[c].x, o.y + f * po[c].y, o.z + f * po[c].z, o.w + f * po[c].w);
          l += f * ml[c].y;
        }
    }
  }
};

// The last part of a (row, slice of the dims) to finish stitches them, in key order.
// T threads take every T-th part of four dims of a head each, so that one round
// of loads reaches all parts (one thread each: 3 of them in turn for 24 parts).
__device__ __forceinline__ void stitch_parts(const Args& a, size_t row, size_t part0, int rank, int slices, int nparts,
                                             int* last) {
  __syncthreads();
  if (threadIdx.x == 0) *last = arrive_last(&a.counters[row * slices + rank], nparts);
  __syncthreads();
  if (!*last) return;
  const int quads = kD / 4 / slices, items = a.group * quads;
  int T = 1;
  while (T * Joined::kBatch < nparts && 2 * T * items <= kWarps * 32) T *= 2;  // at most 32: 4 items at least
  const int sub = threadIdx.x & (T - 1);
  for (int i0 = 0; i0 < items; i0 += kWarps * 32 / T) {
    const int i = i0 + threadIdx.x / T, at = min(i, items - 1);
    const int h = at / quads, d = (rank * quads + at % quads) * 4;
    Joined sum;
    sum.add(sub < nparts ? (nparts - sub + T - 1) / T : 0, [&](int p, float2& ml, float4& o) {
      const size_t from = part0 + sub + p * T;
      ml = __ldcg(reinterpret_cast<const float2*>(a.part_ml) + (from * slices + rank) * a.group + h);
      o = __ldcg(reinterpret_cast<const float4*>(a.part_o + (from * a.group + h) * kD + d));
    });
    for (int x = 1; x < T; x <<= 1) {
      const float top = fmaxf(sum.m, __shfl_xor_sync(0xffffffffu, sum.m, x)), f = ex2(sum.m - top);
      sum.m = top;
      sum.l *= f;
      sum.o = make_float4(sum.o.x * f, sum.o.y * f, sum.o.z * f, sum.o.w * f);
      sum.l += __shfl_xor_sync(0xffffffffu, sum.l, x);
      sum.o.x += __shfl_xor_sync(0xffffffffu, sum.o.x, x);
      sum.o.y += __shfl_xor_sync(0xffffffffu, sum.o.y, x);
      sum.o.z += __shfl_xor_sync(0xffffffffu, sum.o.z, x);
      sum.o.w += __shfl_xor_sync(0xffffffffu, sum.o.w, x);
    }
    if (sub == 0 && i < items) store_out(a, row * a.group + h, d, sum.o, sum.l);
  }
}

// What one cluster (or single CTA) takes of the rows of a kv head.
struct Share {
  int b;            // sequence, -1: nothing
  int unit0, part;  // the sequence's first cluster, and which one of them this is
  int split_tiles;  // blocks per CTA
  int len;          // the sequence's, as given
};
// Cluster `unit` of a.units: sequences get clusters by their blocks, with the
// smallest split (of kMinSplit blocks or more) at which they suffice.  Every warp
// works it out for itself.
__device__ __forceinline__ Share share_of(const Args& a, int unit, int slices, int lane) {
  if (a.num_seqs == 1) {
    const int len = a.seq_lens[0], all = a.units * slices;
    return Share{0, 0, unit, max((int)kMinSplit, (keys_of(a, len).tiles + all - 1) / all), len};
  }
  auto tiles = [&](int i) { return i < a.num_seqs ? keys_of(a, a.seq_lens[i]).tiles : 0; };
  int total = 0;
#pragma unroll 1
  for (int i = lane; i < a.num_seqs; i += 32) total += tiles(i);
  total = __reduce_add_sync(0xffffffffu, total);  // below 2^31 (plan)
  unsigned t = max((unsigned)kMinSplit, (unsigned)(total + a.units * slices - 1) / (a.units * slices));
  auto clusters = [&](int i) -> unsigned {
    const unsigned n = tiles(i);
    return i >= a.num_seqs ? 0 : n <= kLoneRow ? 1 : (n + t * slices - 1) / (t * slices);
  };
#pragma unroll 1
  while (true) {  // ends: with t the longest row's blocks, a.units >= num_seqs clusters suffice
    unsigned n = 0;
#pragma unroll 1
    for (int i = lane; i < a.num_seqs; i += 32) n += clusters(i);
    n = __reduce_add_sync(0xffffffffu, n);
    if (n <= (unsigned)a.units) break;
    t = max(t + t / 16 + 1, (unsigned)((float)t * (float)n / (float)a.units));
  }
  int before = 0;
#pragma unroll 1
  for (int i0 = 0; i0 < a.num_seqs; i0 += 32) {
    const int mine = clusters(i0 + lane);
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const int first = before + upto - mine;
    const unsigned at = __ballot_sync(0xffffffffu, unit >= first && unit < first + mine);
    if (at != 0) {
      const int from = __ffs(at) - 1, unit0 = __shfl_sync(0xffffffffu, first, from);
      return Share{i0 + from, unit0, unit - unit0, (int)t, a.seq_lens[i0 + from]};
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return Share{-1, 0, 0, (int)t, 0};
}

// ---- few rows: one CTA per split --------------------------------------------------
template <bool CAP>
__global__ void __launch_bounds__(kWarps * 32, kCtasPerSm) splits_kernel(const Args a) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float sm_m[kWarps][8];
  __shared__ float sm_l[kWarps][8];
  __shared__ __align__(8) float cta_ml[8][2];
  __shared__ int sm_last;
  __shared__ __align__(8) int sm_blk[kWarps][kBlkRing];
  if (!a.inputs_stable) pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int Hkv = a.num_kv_heads, group = a.group;
  const int slices = (int)cg::this_cluster().num_blocks();
  const int split0 = blockIdx.x / slices * slices;  // the cluster's first CTA
  const Share sh = a.units != 0 ? share_of(a, split0 / slices, slices, lane)
                                : Share{(int)blockIdx.z, 0, split0 / slices, a.split_tiles, a.seq_lens[blockIdx.z]};
  if (sh.b < 0) return;
  const int g = blockIdx.y, b = sh.b, part = sh.part, split_tiles = sh.split_tiles;
  const int split = part * slices + (blockIdx.x - split0);
  const size_t row = (size_t)b * Hkv + g;
  // of the row's first part in the workspace
  const size_t part0 = a.units != 0 ? (size_t)g * a.units + sh.unit0 : row * a.max_parts;

  const Keys seq = keys_of(a, sh.len);
  if (sh.len != seq.seq_len && split == 0 && g == 0 && threadIdx.x == 0) report(a.status, DOE_DEVICE_ERR_LENGTH);
  const int nsplits = a.units != 0 && seq.tiles <= kLoneRow ? 1 : max(1, (seq.tiles + split_tiles - 1) / split_tiles);
  const int nparts = (nsplits + slices - 1) / slices;
  if (part >= nparts) return;             // the whole cluster; a split past the last joins with nothing
  if (nsplits == 1 && split != part * slices) return;  // nothing to join
  const int tile_begin = split * split_tiles;
  const int tile_end = nsplits == 1 ? seq.tiles : min(seq.tiles, tile_begin + split_tiles);
  const int span = tile_end - tile_begin - warp;
  const Stretch w = {b, g, seq.seq_len, seq.min_key, seq.origin + tile_begin + warp,
                     span > 0 ? (span + kWarps - 1) / kWarps : 0, 0, nsplits == 1};
  Walker<CAP, kWarps> walker(a, sm_blk[warp], ring + warp * kWarpBytes, lane);
  // the first copies go out before the query work, and before griddepcontrol.wait
  // when the caller vouches for the inputs
  walker.start(w);
  if (a.inputs_stable) pdl_wait();
  pdl_trigger();
  Sums sums;
  walker.walk(w, sums);

  // ---- join the warps: O staged in the ring's first slots ---------------------------
  if (r == 0)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      sm_m[warp][2 * t + j] = sums.m[j];
      sm_l[warp][2 * t + j] = sums.l[j];
    }
  float* my_o = reinterpret_cast<float*>(ring + warp * kWarpBytes);  // [8][128]
  walker.each(sums, [&](int j, int d, const float4& v) {
    *reinterpret_cast<float4*>(my_o + (2 * t + j) * kD + d) = v;
  });
  __syncthreads();
  const size_t part_row = part0 + part;
  float* cta_o = reinterpret_cast<float*>(ring);  // [8][128], over the first warp's
  for (int i = threadIdx.x; i < group * (kD / 4); i += kWarps * 32) {
    const int h = i / (kD / 4), d = i % (kD / 4) * 4;
    float M = kNone, L = 0.0f;
    float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < kWarps; ++c) M = fmaxf(M, sm_m[c][h]);
#pragma unroll
    for (int c = 0; c < kWarps; ++c) {
      const float f = ex2(sm_m[c][h] - M);
      const float4 o = *reinterpret_cast<const float4*>(ring + c * kWarpBytes + (h * kD + d) * 4);
      O = make_float4(O.x + f * o.x, O.y + f * o.y, O.z + f * o.z, O.w + f * o.w);
      L += f * sm_l[c][h];
    }
    if (nsplits == 1) {
      store_out(a, row * group + h, d, O, L);
    } else {
      float* ml = slices == 1 ? a.part_ml + (part_row * group + h) * 2 : cta_ml[h];
      // over what only this thread has read
      *reinterpret_cast<float4*>(slices == 1 ? a.part_o + (part_row * group + h) * kD + d : cta_o + h * kD + d) = O;
      if (d == 0) {
        ml[0] = M;
        ml[1] = L;
      }
    }
  }
  if (nsplits == 1) return;

  // ---- join the cluster: this CTA its slice of the dims -------------------------------
  const int quads = kD / 4 / slices;
  int rank = 0;
  if (slices > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    rank = (int)cluster.block_rank();
    cluster.sync();
    for (int i = threadIdx.x; i < group * quads; i += kWarps * 32) {
      const int h = i / quads, d = (rank * quads + i % quads) * 4;
      Joined sum;
      sum.add(slices, [&](int c, float2& ml, float4& o) {
        ml = *reinterpret_cast<const float2*>(cluster.map_shared_rank(cta_ml[h], c));
        o = *reinterpret_cast<const float4*>(cluster.map_shared_rank(cta_o, c) + h * kD + d);
      });
      if (nparts == 1) {
        store_out(a, row * group + h, d, sum.o, sum.l);
      } else {
        *reinterpret_cast<float4*>(a.part_o + (part_row * group + h) * kD + d) = sum.o;
        if (i % quads == 0)
          *reinterpret_cast<float2*>(a.part_ml + ((part_row * slices + rank) * group + h) * 2) =
              make_float2(sum.m, sum.l);
      }
    }
    cluster.sync();  // this CTA has read the others' parts
  }
  if (nparts > 1) stitch_parts(a, row, part0, rank, slices, nparts, &sm_last);
}

// ---- many rows: pieces of one list, a warp each -------------------------------------
template <bool CAP>
__global__ void __launch_bounds__(kWarps * 32, kCtasPerSm) pieces_kernel(const Args a) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(8) int sm_blk[kWarps][kBlkRing];
  __shared__ int sm_end[kMaxListSeqs];  // entries of sequences 0..b
  __shared__ int sm_len[kMaxListSeqs];
  __shared__ int sm_sum[kWarps];
  if (!a.inputs_stable) pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  const int Hkv = a.num_kv_heads, group = a.group;

  // the list has the sequences one after another, each as kRowCost entries for
  // its fixed cost and one per block (an empty one as if it had one, so that
  // somebody writes its zeros)
  {
    const int per = (a.num_seqs + kWarps * 32 - 1) / (kWarps * 32), b0 = threadIdx.x * per;
    int sum = 0;
    for (int i = b0; i < min(b0 + per, a.num_seqs); ++i) {
      const int raw = a.seq_lens[i];
      const Keys s = keys_of(a, raw);
      if (raw != s.seq_len && blockIdx.x == 0) report(a.status, DOE_DEVICE_ERR_LENGTH);
      sum += kRowCost + max(1, s.tiles);
      sm_end[i] = sum;
      sm_len[i] = raw;
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
  }
  // An item is a piece of one kv head, the head fastest
  const int total = sm_end[a.num_seqs - 1];  // below 2^29 (plan)
  const int most = (int)gridDim.x * kWarps / Hkv;                   // pieces (at least one: plan)
  const int size = max(kMinPiece, (total + most - 1) / most);        // of a piece
  const int items = (total + size - 1) / size * Hkv;
  int item = blockIdx.x * kWarps + warp;
  if (item >= items) return;

  int at = 0, end = 0, b = 0, g = 0;  // what is left of the piece, its sequence and head
  auto seq_size = [&](int s) { return sm_end[s] - (s ? sm_end[s - 1] : 0); };
  auto seq_of = [&](int x, int lo) {  // the sequence that holds entry x, at least lo
    int hi = a.num_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (sm_end[mid] > x) hi = mid;
      else lo = mid + 1;
    }
    return lo;
  };
  auto open_piece = [&]() {
    const int piece = item / Hkv;
    g = item - piece * Hkv;
    at = piece * size;
    end = min(total, at + size);
    b = seq_of(at, b);
    // an end inside a sequence's fixed cost leaves that sequence to the next piece
    const int s = seq_of(end - 1, b), over = end - (sm_end[s] - seq_size(s));
    if (over <= kRowCost) end -= over;
  };
  auto take = [&]() {  // the piece's next stretch
    if (at >= sm_end[b]) ++b;
    const int row_size = seq_size(b), row_at = sm_end[b] - row_size;
    const Keys seq = keys_of(a, sm_len[b]);
    const int tile_begin = max(0, at - row_at - kRowCost);
    at = min(end, row_at + row_size);
    const int tile_end = min(at - row_at - kRowCost, seq.tiles);
    return Stretch{b, g, seq.seq_len, seq.min_key, seq.origin + tile_begin, max(0, tile_end - tile_begin), row_at,
                   tile_begin == 0 && at == row_at + row_size};
  };

  Walker<CAP, 1> walker(a, sm_blk[warp], ring + warp * kWarpBytes, lane);
  open_piece();
  Stretch cur = take();
  walker.start(cur);
  if (a.inputs_stable) pdl_wait();
  pdl_trigger();
  int cut_row[2] = {-1, -1}, cut_at[2] = {0, 0};   // rows that the piece holds a part of
  bool first = true;                               // the piece's first stretch
  while (true) {
    Sums sums;
    walker.walk(cur, sums);

    // the next stretch's first copies go out before this one's results
    const Stretch done = cur;
    const bool more = at < end;
    if (more) {
      cur = take();
      walker.start(cur);
    }

    const size_t row = (size_t)done.b * Hkv + done.g;
    if (done.whole) {
      walker.each(sums, [&](int j, int d, const float4& v) {
        if (2 * t + j < group) store_out(a, row * group + 2 * t + j, d, v, sums.l[j]);
      });
    } else {
      const size_t part = 2 * (size_t)item + (first ? 0 : 1);
      walker.each(sums, [&](int j, int d, const float4& v) {
        if (2 * t + j < group) *reinterpret_cast<float4*>(a.part_o + (part * group + 2 * t + j) * kD + d) = v;
      });
      if (r == 0)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (2 * t + j < group)
            *reinterpret_cast<float2*>(a.part_ml + (part * group + 2 * t + j) * 2) = make_float2(sums.m[j], sums.l[j]);
      if (first) {
        cut_row[0] = (int)row;
        cut_at[0] = done.row_at;
      } else {
        cut_row[1] = (int)row;
        cut_at[1] = done.row_at;
      }
    }
    first = false;
    if (!more) break;
  }

  // ---- the last part of a row to finish stitches them, in key order ------------------
  if (cut_row[0] < 0 && cut_row[1] < 0) return;
  __syncwarp();
  const int e = lane & 1;  // lanes 0 and 1 take a row each
  const int my_row = cut_row[e], my_at = cut_at[e];
  int c0 = 0, n = 0, last = 0;
  if (my_row >= 0) {
    c0 = (my_at + kRowCost) / size;
    n = (my_at + seq_size(my_row / Hkv) - 1) / size - c0 + 1;
    if (lane < 2) last = arrive_last(&a.counters[my_row], n);
  }
  __syncwarp();
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    if (!__shfl_sync(0xffffffffu, last, i)) continue;
    const int from0 = __shfl_sync(0xffffffffu, c0, i), parts = __shfl_sync(0xffffffffu, n, i);
    const int row = cut_row[i];
    // in its first piece, a row that another one precedes is the second part
    const int second = from0 * size < cut_at[i] ? 1 : 0;
    auto part_at = [&](int p, int h) {
      return (2 * ((size_t)(from0 + p) * Hkv + g) + (p == 0 ? second : 0)) * group + h;
    };
    for (int h0 = 0; h0 < group; h0 += 4) {  // four heads together: one after another took 16 % more at 30 parts
      float M[4], L[4];
      float4 O[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        M[j] = kNone;
        L[j] = 0.0f;
        O[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
      for (int p0 = 0; p0 < parts; p0 += 32) {  // lane p weighs part p0 + p
        float weight[4];
        float2 ml[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          ml[j] = p0 + lane < parts ? __ldcg(reinterpret_cast<const float2*>(a.part_ml) +
                                             part_at(p0 + lane, min(h0 + j, group - 1)))
                                    : make_float2(kNone, 0.0f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float top = fmaxf(M[j], warp_max(ml[j].x)), f = ex2(M[j] - top);
          weight[j] = ex2(ml[j].x - top);
          L[j] = L[j] * f + warp_sum(weight[j] * ml[j].y);
          O[j] = make_float4(O[j].x * f, O[j].y * f, O[j].z * f, O[j].w * f);
          M[j] = top;
        }
        constexpr int kBatch = 6;  // parts whose loads are in flight together
        const int some = min(32, parts - p0);
        for (int q = 0; q < some; q += kBatch) {
          float4 o[kBatch][4];
#pragma unroll
          for (int c = 0; c < kBatch; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              o[c][j] = __ldcg(reinterpret_cast<const float4*>(
                  a.part_o + part_at(p0 + min(q + c, some - 1), min(h0 + j, group - 1)) * kD + 4 * lane));
#pragma unroll
          for (int c = 0; c < kBatch; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float w = __shfl_sync(0xffffffffu, weight[j], (q + c) & 31);
              if (q + c < some)
                O[j] = make_float4(O[j].x + w * o[c][j].x, O[j].y + w * o[c][j].y, O[j].z + w * o[c][j].z,
                                   O[j].w + w * o[c][j].w);
            }
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (h0 + j < group) store_out(a, (size_t)row * group + h0 + j, 4 * lane, O[j], L[j]);
    }
  }
}

template <typename Kernel>
int launch_one(Kernel kernel, std::atomic<bool> (&attr)[kMaxDevices], const Args& a, dim3 grid, unsigned slices,
               cudaStream_t st) {
  const int rc = once_per_device(attr, [&] {
    return cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem),
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
  return cuda_status(cudaLaunchKernelEx(&cfg, kernel, a), "paged_decode_int4");
}

template <bool CAP>
int launch_cap(const Args& a, bool list, dim3 grid, unsigned slices, cudaStream_t st) {
  static std::atomic<bool> attr[2][kMaxDevices];
  return list ? launch_one(pieces_kernel<CAP>, attr[0], a, grid, slices, st)
              : launch_one(splits_kernel<CAP>, attr[1], a, grid, slices, st);
}

// How a launch is cut, and the sizes that follow.
struct Plan {
  bool list;                     // pieces of one list; else splits
  uint64_t split_tiles, slices;  // splits: blocks per split, splits per cluster
  uint64_t units;                // splits that follow the lengths: clusters per kv head
  uint64_t max_parts, grid;      // splits: parts per row; CTAs (per row, or per kv head)
  uint64_t slots;                // parts in the workspace (whatever the window, which its size query lacks)
};

// `tiles`: the most blocks of a row that can be read (its block-table row, or the
// window).  In order (times of this rule against the other one):
//  - a given split_pages: splits of that length;
//  - rows for every SM, of kShortRow blocks at most: one CTA each, nothing to join (32
//    x 8 rows of 1024 tokens 16.7 us, of 2048 27; as a list 23 and 30);
//  - rows below a seventh of the resident warps: splits by the lengths (24 x 8
//    rows of 1k-8k 37.7 us, as a list 39.8; 16 x 8 of 1k-16k 43, 47.  From there
//    on the list: 32 x 8 of 500-16k 71 us, 84 in splits; 32 x 8 of 8k-32k 145, 174).
//    Their sum is what is resident at once: 3 CTAs per SM, or 384 in clusters of 8, which
//    not every SM's place can join (1 x 130001 tokens, 2 kv heads: 27 us with 444).
//    Clusters where a row gets more than 16 splits (that row without: 27 us in
//    pairs, 20 in eights).  Splits that follow the table's width instead of the
//    lengths cost 63 us against 19 for 4 x 8192 tokens in tables for 131072;
//  - else the list, if the device can count its entries.
Plan plan(uint64_t num_seqs, uint64_t kv_heads, uint64_t max_tiles, uint64_t tiles_per_page, uint64_t split_pages,
          uint64_t window) {
  Plan p = {};
  const uint64_t rows = num_seqs * kv_heads, sms = (uint64_t)num_sms(), ctas = sms * kCtasPerSm;
  const uint64_t tiles = window != 0 && window / 16 + 2 < max_tiles ? window / 16 + 2 : max_tiles;
  const bool counted = num_seqs * (max_tiles + kRowCost) <= 0x1fffffffull;  // the device's sums of blocks
  uint64_t t = split_pages * tiles_per_page;
  const bool short_rows = t == 0 && rows >= sms && tiles <= kShortRow;
  if (short_rows) {
    t = tiles;
  } else if (t == 0 && rows * kListRows < ctas * kWarps && counted) {
    p.slices = max_tiles > 16 * kMinSplit && rows * 16 < sms * 13 / 5 ? 8 : 1;
    const uint64_t fill = p.slices > 1 ? sms * 13 / 5 / p.slices : ctas;
    // no more than the rows can use at all, and one for every row
    const uint64_t most = max_tiles <= kLoneRow ? 1 : (max_tiles + kMinSplit * p.slices - 1) / (kMinSplit * p.slices);
    p.units = std::max(num_seqs, std::min(fill / kv_heads, num_seqs * most));
    p.max_parts = 2;
    p.grid = p.units * p.slices;
    p.slots = p.units * kv_heads;
    return p;
  } else if (t == 0 && num_seqs <= kMaxListSeqs && kv_heads <= ctas * kWarps && counted) {
    p.list = true;
    p.slices = 1;
    p.max_parts = 2;
    p.grid = ctas;
    p.slots = 2 * ctas * kWarps;
    return p;
  } else if (t == 0) {
    t = rows >= sms ? tiles : (tiles * rows + sms - 1) / sms;
    if (t < kMinSplit) t = kMinSplit;
    p.slots = rows >= sms ? rows : sms + rows;
  } else {
    p.slots = rows * ((max_tiles + t - 1) / t);
  }
  p.split_tiles = t < tiles ? t : tiles;
  const uint64_t splits = (tiles + p.split_tiles - 1) / p.split_tiles;
  p.slices = splits > 16 ? 8 : 1;
  p.max_parts = (splits + p.slices - 1) / p.slices;
  p.grid = p.max_parts * p.slices;
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
  const Plan pl = plan(num_seqs ? num_seqs : 1, Hkv, max_tiles, tpp, split_pages, opts ? opts->sliding_window : 0);
  // The counters come first, in a region of one size for all but huge batches, so
  // that decodes of any shapes can share a workspace whose counters stay zero; a
  // huge batch's, which others' parts overwrite, are cleared by every launch.  A
  // part has O and, for each of up to 8 slices, (m, l) per head.
  const uint64_t ctr_bytes = (rows * 8 * sizeof(unsigned) + kCounterBytes - 1) / kCounterBytes * kCounterBytes;
  const uint64_t parts = pl.slots * group;
  const uint64_t ws = ctr_bytes + parts * (kD + 2 * 8) * sizeof(float);
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
  for (const void* p : {(const void*)kv->k_pool, (const void*)kv->v_pool, q, (const void*)launch->workspace, (const void*)out})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) {
      set_op_error("doe_paged_decode: pools, q, out and the workspace must be 16-byte aligned");
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
  a.counters = static_cast<unsigned*>(launch->workspace);
  a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(launch->workspace) + ctr_bytes);
  a.part_ml = a.part_o + parts * kD;
  a.status = launch->status;
  a.freq_cis = opts ? opts->freq_cis : nullptr;
  a.rope_positions = opts ? (int)opts->rope_positions : 0;
  a.window = opts ? (int)(opts->sliding_window > 0x7fffffffu ? 0x7fffffffu : opts->sliding_window) : 0;
  // A score is at most 128 * 65504^2 |scale| < 2^39 |scale|, and tanh(y) is y within 2^-25 below y =
  // 2^-12: a cap from 2^51 |scale| on changes nothing.
  a.softcap = opts && opts->attn_softcap < 0x1p51f * std::fabs(scale) ? opts->attn_softcap : 0.0f;
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
  a.units = (int)pl.units;
  a.out_bf16 = (opts && (opts->flags & DOE_DECODE_OUT_BF16)) ? 1 : 0;
  a.inputs_stable = (opts && (opts->flags & DOE_DECODE_INPUTS_STABLE)) ? 1 : 0;
  cudaStream_t st = static_cast<cudaStream_t>(launch->stream);
  const bool zeroed = opts && (opts->flags & DOE_DECODE_COUNTERS_ZEROED) && ctr_bytes == kCounterBytes;
  if ((pl.list || pl.max_parts > 1) && !zeroed) {
    const int rc =
        cuda_status(cudaMemsetAsync(a.counters, 0, rows * pl.slices * sizeof(unsigned), st), "cudaMemsetAsync(split counters)");
    if (rc != DOE_OK) return rc;
  }
  const dim3 grid = pl.list ? dim3((unsigned)pl.grid) : dim3((unsigned)pl.grid, Hkv, pl.units != 0 ? 1 : num_seqs);
  return a.softcap > 0.0f ? launch_cap<true>(a, pl.list, grid, (unsigned)pl.slices, st)
                          : launch_cap<false>(a, pl.list, grid, (unsigned)pl.slices, st);
}

}  // namespace doe
