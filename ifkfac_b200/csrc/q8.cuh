// The 8-bit row format (include/ifk.h, ifk_q8_pitch): a group of 32 columns of a
// row shares the scale 2^e, stored as the byte e + 127; a value is code * 2^e.
#pragma once

#include "ifk_common.cuh"

namespace ifk {
namespace q8 {

constexpr int GROUP = IFK_Q8_GROUP;

__host__ __device__ inline int64_t pitch(int64_t n) { return cdiv(n, GROUP) * GROUP; }

// The group's scale byte from the largest |x| of the group as fp32 bits.  The
// exponent field is floor(log2 |x|) + 127, so the byte is that field less 6; 255
// stands for a NaN or an infinity in the group.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  const int E = (int)(amax_bits >> 23);
  if (E == 255) return 255u;
  return (uint32_t)mx(E - 6, 1);
}
// 2^-e and 2^e of a finite group's scale byte (1 .. 248: both are normal numbers).
__device__ __forceinline__ float inv_scale(uint32_t s) { return __uint_as_float((254u - s) << 23); }
// 2^e, or +inf for byte 255, whose codes are 0: 0 * inf reads as NaN.
__device__ __forceinline__ float scale_of(uint32_t s) { return __uint_as_float(s << 23); }

// Whether a code of the group can round to 128 and has to be clipped: the largest |x| 2^-e is 127.5 or more.
__device__ __forceinline__ bool may_clip(uint32_t amax_bits) { return (amax_bits & 0x007fffffu) >= 0x007f0000u; }

// code of x as the low byte of the fp32 bits of code + 1.5 * 2^23: x 2^-e is exact, and the addition rounds
// to the nearest integer, ties to even.
__device__ __forceinline__ uint32_t code_bits(float x, float inv) {
  return __float_as_uint(fmaf(x, inv, 12582912.f));
}
__device__ __forceinline__ uint32_t code_bits_clipped(float x, float inv) {
  return __float_as_uint(fminf(fmaxf(x * inv, -127.f), 127.f) + 12582912.f);
}

// The value of one of four packed codes: the byte with its sign bit flipped is
// code + 128, placed under the exponent of 2^23.
__device__ __forceinline__ float value_of(uint32_t flipped, int byte, float scale) {
  const float u = __uint_as_float(__byte_perm(flipped, 0x4b000000u, 0x7540 | byte));
  return (u - 8388736.f) * scale;
}

}  // namespace q8

}  // namespace ifk
