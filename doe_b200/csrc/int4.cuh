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

__device__ __forceinline__ float div7(float amax) { return __fdiv_rn(amax, 7.0f); }

// clamp(rint(x / s), -7, 7) + 8 for f16 values x and an f16 scale s > 0, from
// the correctly rounded reciprocal rs: the same quotient as quantize_s8, whose
// argument that it rounds as the IEEE quotient does holds for any f16 operands
// with |x / s| <= 127.  Adding 1.5 * 2^23 + 8 rounds half to even (8 is even).
__device__ __forceinline__ uint32_t quantize_u4(float x, float s, float rs) {
  const float y0 = x * rs;
  const float y = fmaf(fmaf(-y0, s, x), rs, y0);
  const float c = fminf(fmaxf(y, -7.0f), 7.0f);
  return __float_as_uint(__fadd_rn(c, 12582920.0f)) & 15u;
}

}  // namespace doe
