// int4.cuh -- the 4-bit KV block shared by the append, read and decode kernels.
//
// A row of head_dim 128 is held in 4 groups of 32 dims, each with an f16 scale:
//   s = f16(max|x| / 7),  q = clamp(rint(x / s), -7, 7)  (0 when s == 0),
// stored as n = q + 8 (1..15), so a value is (n - 8) * s.  f16 scales and 15
// levels keep the definition of the int8 cache (f16(max|x| / 127), symmetric);
// a scale per 32 dims instead of per row costs 8 bytes in 72 and holds the
// error to the group's own maximum.
//
// 16 tokens of one kv head are one block of 1152 bytes: 1024 bytes of codes in
// the order the decode's fragments read them, then 128 bytes of scales, so a
// block is one contiguous copy and every fragment read one 16-byte load.
//   K codes: word [token][t][group] (t = 0..3): dims 32 group + 8 t + 2 i in
//            bits 4 i of the low half and the odd dims + 1 in the high half:
//            (w >> 4 i) & 0x000f000f is a pair of adjacent dims;
//   V codes: 16-bit half [token >> 3][g][(token >> 1) & 3][group][token & 1]
//            (g = 0..7): dims 32 group + 4 g + i in bits 4 i: the same mask
//            gives one dim of two adjacent tokens;
//   K scales [token][group], V scales [token >> 1][group][token & 1], f16.
// A row of one token is 64 bytes of whole 16-bit halves in both, so tokens are
// appended one at a time without reading the block back.
#pragma once

#include "common.cuh"

namespace doe {

constexpr int kI4Codes = 1024;
constexpr int kI4Block = 1152;

// amax / 7 without an IEEE division: one residual correction of amax * RN(1/7)
// (Markstein's method).  For every finite f16 amax >= 0 it is the correctly
// rounded f32 quotient (checked for all of them against f32 division).
__device__ __forceinline__ float div7(float amax) {
  constexpr float kInv7 = 0x1.24924ap-3f;  // RN_f32(1 / 7)
  const float q0 = amax * kInv7;
  return fmaf(fmaf(-q0, 7.0f, amax), kInv7, q0);
}
// About 1 / s, and 0 for 0 (so that a row of zeros gets the code of 0).
__device__ __forceinline__ float inverse_of(float s) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(s));
  return s > 0.0f ? r : 0.0f;
}

// rint(x / s) of two f16 values, as words whose low nibble is the code, n =
// rint(x / s) + 8.  y0 = x rs, y = y0 + (x - y0 s) rs is the quotient up to an
// error far below its distance from every half-integer (which is 0 or at least
// 2^-14, see quantize_s8), and in a tie exactly k + 1/2, for any rs within a few
// ulps of 1 / s.  Adding 1.5 * 2^23 + 8 rounds half to even (8 is even).  With s =
// f16(max|x| / 7) normal, |x / s| <= 7 / (1 - 2^-11) rounds to 7 at most; a
// subnormal s may be rounded down by more, then CLAMP.
template <bool CLAMP>
__device__ __forceinline__ uint2 quantize_u4x2(float2 x, float s, float rs) {
  const float2 rs2 = make_float2(rs, rs);
  const float2 y0 = fmul2(x, rs2);
  float2 y = ffma2(ffma2(y0, make_float2(-s, -s), x), rs2, y0);
  if (CLAMP) y = make_float2(fminf(fmaxf(y.x, -7.0f), 7.0f), fminf(fmaxf(y.y, -7.0f), 7.0f));
  const float2 c = fadd2(y, make_float2(12582920.0f, 12582920.0f));
  return make_uint2(__float_as_uint(c.x), __float_as_uint(c.y));
}
__device__ __forceinline__ uint2 quantize_u4x2(float2 x, float s, float rs) {
  return s >= 0x1p-14f ? quantize_u4x2<false>(x, s, rs) : quantize_u4x2<true>(x, s, rs);
}
// Four such words' codes, the first lowest, in the low 16 bits of the result (the
// other bits are anything): the words are 0x4b400008 + q, and the multiples of
// 16 of their upper bits leave the low 16 bits alone but for 8 in each nibble.
__device__ __forceinline__ uint32_t pack_u4x4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return ((d * 16u + c) * 16u + b) * 16u + a;
}

}  // namespace doe
