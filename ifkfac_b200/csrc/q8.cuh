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

// Eight neighbouring columns of a row from column c on; columns at or past n read
// as 0.  vec: the row is 16-byte aligned (c is a multiple of 8).
__device__ __forceinline__ void load8(const float* row, int64_t c, int64_t n, bool vec, float (&v)[8]) {
  if (vec && c + 8 <= n) {
    const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < n ? row[c + i] : 0.f;
  }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* row, int64_t c, int64_t n, bool vec, float (&v)[8]) {
  if (vec && c + 8 <= n) {
    const uint4 a = *reinterpret_cast<const uint4*>(row + c);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < n ? __bfloat162float(row[c + i]) : 0.f;
  }
}
__device__ __forceinline__ void store8(float* row, int64_t c, int64_t n, bool vec, const float (&v)[8]) {
  if (vec && c + 8 <= n) {
    *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(row + c + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < n) row[c + i] = v[i];
  }
}
__device__ __forceinline__ void store8(__nv_bfloat16* row, int64_t c, int64_t n, bool vec, const float (&v)[8]) {
  if (vec && c + 8 <= n) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
    *reinterpret_cast<uint4*>(row + c) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < n) row[c + i] = __float2bfloat16_rn(v[i]);
  }
}

// Rows of a matrix of element type T: 16-byte accesses at columns that are multiples of 8.
template <typename T>
inline bool rows_aligned(const T* p, int64_t ld) {
  return (((uintptr_t)p) & 15) == 0 && (ld * (int64_t)sizeof(T)) % 16 == 0;
}

}  // namespace ifk
