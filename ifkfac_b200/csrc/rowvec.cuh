// V neighbouring columns of a row in a thread: one access of V elements where the row is
// aligned for it, one at a time at a ragged end.
#pragma once

#include "ifk_common.cuh"
#include "q8.cuh"

namespace ifk {

template <typename T, int V>
struct Raw;  // V elements as they are in memory
template <> struct Raw<float, 4> { float4 r; };
template <> struct Raw<float, 1> { float r; };
template <> struct Raw<__nv_bfloat16, 16> { uint4 r, q; };
template <> struct Raw<__nv_bfloat16, 8> { uint4 r; };
template <> struct Raw<__nv_bfloat16, 4> { uint2 r; };
template <> struct Raw<__nv_bfloat16, 1> { __nv_bfloat16 r; };

// Two fp32 values in a 64-bit register: one instruction does both, each rounded on its own.
struct F2 {
  uint64_t r;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 q;
  asm("mov.b64 %0, {%1, %2};" : "=l"(q.r) : "f"(a), "f"(b));
  return q;
}
__device__ __forceinline__ F2 f2(float a) { return f2(a, a); }
__device__ __forceinline__ void split(F2 q, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(q.r));
}
__device__ __forceinline__ float sum(F2 q) {
  float a, b;
  split(q, a, b);
  return a + b;
}
__device__ __forceinline__ F2 add(F2 a, F2 b) {
  F2 q;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(q.r) : "l"(a.r), "l"(b.r));
  return q;
}
__device__ __forceinline__ F2 mul(F2 a, F2 b) {
  F2 q;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(q.r) : "l"(a.r), "l"(b.r));
  return q;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 q;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(q.r) : "l"(a.r), "l"(b.r), "l"(c.r));
  return q;
}
template <int N>
__device__ __forceinline__ void pairs(const float (&v)[2 * N], F2 (&q)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) q[i] = f2(v[2 * i], v[2 * i + 1]);
}
template <int N>
__device__ __forceinline__ void singles(const F2 (&q)[N], float (&v)[2 * N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) split(q[i], v[2 * i], v[2 * i + 1]);
}

__device__ __forceinline__ void bf16x2(uint32_t w, float& a, float& b) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void unpack(const Raw<float, 4>& q, float (&v)[4]) {
  v[0] = q.r.x;
  v[1] = q.r.y;
  v[2] = q.r.z;
  v[3] = q.r.w;
}
__device__ __forceinline__ void unpack(const Raw<float, 1>& q, float (&v)[1]) { v[0] = q.r; }
__device__ __forceinline__ void unpack(const Raw<__nv_bfloat16, 1>& q, float (&v)[1]) { v[0] = __bfloat162float(q.r); }
__device__ __forceinline__ void unpack(const Raw<__nv_bfloat16, 4>& q, float (&v)[4]) {
  bf16x2(q.r.x, v[0], v[1]);
  bf16x2(q.r.y, v[2], v[3]);
}
__device__ __forceinline__ void unpack(const Raw<__nv_bfloat16, 16>& q, float (&v)[16]) {
  bf16x2(q.r.x, v[0], v[1]);
  bf16x2(q.r.y, v[2], v[3]);
  bf16x2(q.r.z, v[4], v[5]);
  bf16x2(q.r.w, v[6], v[7]);
  bf16x2(q.q.x, v[8], v[9]);
  bf16x2(q.q.y, v[10], v[11]);
  bf16x2(q.q.z, v[12], v[13]);
  bf16x2(q.q.w, v[14], v[15]);
}
__device__ __forceinline__ void unpack(const Raw<__nv_bfloat16, 8>& q, float (&v)[8]) {
  bf16x2(q.r.x, v[0], v[1]);
  bf16x2(q.r.y, v[2], v[3]);
  bf16x2(q.r.z, v[4], v[5]);
  bf16x2(q.r.w, v[6], v[7]);
}

// Columns c .. c + V - 1 of the row (c a multiple of V); columns at or past n are 0.  WHOLE: n is a
// multiple of V, so an access is inside the row or past it.
template <typename T, int V, bool WHOLE = false>
__device__ __forceinline__ Raw<T, V> load_raw(const T* row, int c, int n) {
  Raw<T, V> q;
  if (WHOLE) {
    memset(&q, 0, sizeof(q));
    if (c < n) q = *reinterpret_cast<const Raw<T, V>*>(row + c);
    return q;
  }
  if (V == 1) {
    T zero = T(0.f), x = zero;
    if (c < n) x = row[c];
    memcpy(&q, &x, sizeof(T));
    return q;
  }
  if (c + V <= n) return *reinterpret_cast<const Raw<T, V>*>(row + c);
  T e[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    e[i] = T(0.f);
    if (c + i < n) e[i] = row[c + i];
  }
  memcpy(&q, e, sizeof(q));
  return q;
}

// The same columns of a row in shared memory; n is a multiple of V.
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> shared_raw(const uint8_t* row, int c, int n) {
  Raw<T, V> q;
  memset(&q, 0, sizeof(q));
  if (c < n) q = *reinterpret_cast<const Raw<T, V>*>(row + (size_t)c * sizeof(T));
  return q;
}

template <int V, bool WHOLE = false>
__device__ __forceinline__ void store_vec(float* row, int c, int n, const float (&v)[V]) {
  if (V == 4 && (WHOLE || c + 4 <= n)) {
    *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1 % V], v[2 % V], v[3 % V]);
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (c + i < n) row[c + i] = v[i];
}
template <int V, bool WHOLE = false>
__device__ __forceinline__ void store_vec(__nv_bfloat16* row, int c, int n, const float (&v)[V]) {
  if (V > 1 && (WHOLE || c + V <= n)) {
    uint32_t w[(V + 1) / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[(2 * i + 1) % V]);
      w[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
    if (V == 8) *reinterpret_cast<uint4*>(row + c) = make_uint4(w[0], w[1 % ((V + 1) / 2)], w[2 % ((V + 1) / 2)], w[3 % ((V + 1) / 2)]);
    else *reinterpret_cast<uint2*>(row + c) = make_uint2(w[0], w[1 % ((V + 1) / 2)]);
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (c + i < n) row[c + i] = __float2bfloat16_rn(v[i]);
}

// V values of an fp32 vector; the access is whole.
template <int V>
__device__ __forceinline__ void load_f32(const float* p, int c, float (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; j += 4) {
    const float4 q = *reinterpret_cast<const float4*>(p + c + j);
    v[j] = q.x;
    v[(j + 1) % V] = q.y;
    v[(j + 2) % V] = q.z;
    v[(j + 3) % V] = q.w;
  }
}

// V values of a vector of fp32 or bf16 (the weight or bias of a layer norm), or `none` where there is no vector.
template <int V>
__device__ __forceinline__ void load_param(const void* p, bool bf16, float none, int c, int n, float (&v)[V]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = none;
  } else if (bf16) {
    unpack(load_raw<__nv_bfloat16, V>((const __nv_bfloat16*)p, c, n), v);
  } else if (V == 8) {
    float a[4], b[4];
    unpack(load_raw<float, 4>((const float*)p, c, n), a);
    unpack(load_raw<float, 4>((const float*)p, c + 4, n), b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[(4 + i) % V] = b[i];
    }
  } else {
    unpack(load_raw<float, V == 8 ? 4 : V>((const float*)p, c, n), reinterpret_cast<float (&)[V == 8 ? 4 : V]>(v));
  }
}

namespace q8 {

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// The largest |x| of a group whose 32 columns lie V to a lane in 32 / V neighbouring lanes, as bits; a NaN
// comes through as one.
template <int V>
__device__ __forceinline__ uint32_t group_max_bits(const float (&x)[V]) {
  float a = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < V; ++i) a = max_nan(a, fabsf(x[i]));
#pragma unroll
  for (int o = 1; o < GROUP / V; o *= 2) a = max_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
  return __float_as_uint(a) & 0x7fffffffu;
}

// Those of two groups at once, cut to their upper 16 bits: all that the scale and the clipping look at
// (the order of non-negative numbers is that of their upper bits too).
template <int V>
__device__ __forceinline__ void group_max_bits_of_two(const float (&x)[V], const float (&y)[V], uint32_t& mx_x,
                                                      uint32_t& mx_y) {
  float a = fabsf(x[0]), b = fabsf(y[0]);
#pragma unroll
  for (int i = 1; i < V; ++i) {
    a = max_nan(a, fabsf(x[i]));
    b = max_nan(b, fabsf(y[i]));
  }
  uint32_t m = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632) & 0x7fff7fffu;
#pragma unroll
  for (int o = 1; o < GROUP / V; o *= 2) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
  mx_x = m << 16;
  mx_y = m & 0xffff0000u;
}

// V codes of a group with this largest magnitude and scale byte to memory (V-byte aligned).
template <int V>
__device__ __forceinline__ void store_codes(int8_t* p, const float (&x)[V], uint32_t amax_bits, uint32_t s) {
  uint32_t e[V], w[(V + 3) / 4];
  if (s == 255u) {
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = 0u;
  } else if (may_clip(amax_bits)) {
    const float inv = inv_scale(s);
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = code_bits_clipped(x[i], inv);
  } else {
    const float inv = inv_scale(s);
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = code_bits(x[i], inv);
  }
#pragma unroll
  for (int j = 0; j < (V + 3) / 4; ++j)
    w[j] = V == 1 ? e[0]
                  : __byte_perm(__byte_perm(e[(4 * j) % V], e[(4 * j + 1) % V], 0x0040),
                                __byte_perm(e[(4 * j + 2) % V], e[(4 * j + 3) % V], 0x0040), 0x5410);
  constexpr int N = (V + 3) / 4;
  if (V == 16) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1 % N], w[2 % N], w[3 % N]);
  else if (V == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1 % N]);
  else if (V == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
  else *p = (int8_t)w[0];
}

// V packed codes as they are in memory, and their values.
template <int V>
struct Codes {
  uint32_t w[(V + 3) / 4];
};
template <int V>
__device__ __forceinline__ Codes<V> load_codes(const int8_t* p) {
  Codes<V> c;
  if (V == 8) {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    c.w[0] = q.x;
    c.w[(V + 3) / 4 - 1] = q.y;
  } else if (V == 4) {
    c.w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    c.w[0] = (uint8_t)*p;
  }
  return c;
}
template <int V>
__device__ __forceinline__ void values2(const Codes<V>& c, float scale, F2 (&v)[V / 2]) {
  const F2 s = f2(scale), off = f2(-8388736.f);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const uint32_t w = c.w[i / 2] ^ 0x80808080u;
    const float a = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540 | (2 * i & 3)));
    const float b = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540 | ((2 * i + 1) & 3)));
    v[i] = mul(add(f2(a, b), off), s);
  }
}
template <int V>
__device__ __forceinline__ void values(const Codes<V>& c, float scale, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = value_of(c.w[i / 4] ^ 0x80808080u, i & 3, scale);
}

}  // namespace q8

// Whether rows of T with this base and leading dimension allow accesses of V elements.
template <typename T>
inline bool rows_allow(const void* p, int64_t ld, int V) {
  const int64_t b = (int64_t)sizeof(T) * V;
  return (int64_t)((uintptr_t)p % (uintptr_t)b) == 0 && (ld * (int64_t)sizeof(T)) % b == 0;
}

}  // namespace ifk
