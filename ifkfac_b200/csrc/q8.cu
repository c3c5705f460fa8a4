// Activation rows to 8 bits and back (ifk_q8_quantize, ifk_q8_dequantize).
//
// Both are one pass bound by memory: 2 (bf16) or 4 (fp32) bytes an element on one
// side, 1 + 1/32 on the other.  A thread takes V neighbouring columns with one
// access: 16 bytes of the wide side (32 where bf16 rows are quantised: its 16 codes are
// then 16 bytes, too; 37 against 40 us for 16384 x 4096), or one element where its rows
// are not aligned for that (a warp then still covers whole lines).  32 / V neighbouring lanes make a group,
// so the group's maximum is a few shuffles, and a thread has UNROLL accesses in flight
// before it uses the first.  Measured, 16384 x 4096 bf16: to 8 bits 37 us, back 31 to 34 us (203 MB each,
// 5.5 and 6.2 TB/s; a plain copy of this card runs at 6.5).  Small calls are the launch: 2 us on the device.
#include <algorithm>
#include <cstring>

#include "rowvec.cuh"
#include "ifk_internal.h"

namespace ifk {

namespace {

constexpr int THREADS = 256, UNROLL = 4;

// Row i of a call: the row itself, or its entry in the index (-1: out of range).
__device__ __forceinline__ int64_t source_row(int64_t i, const int64_t* ridx, int64_t src_rows, int* status) {
  if (!ridx) return i;
  const int64_t r = ridx[i];
  if (r >= 0 && r < src_rows) return r;
  if (status) *status = IFK_ERR_ARG;
  return -1;
}

// A block takes rpb whole rows of upr accesses; access u of the block belongs to its row u / upr.
struct Units {
  int upr, rpb;
  uint32_t magic;  // ceil(2^32 / upr): u / upr is the high word of u magic, as u upr < 2^32 where rpb > 1
  __device__ __forceinline__ uint32_t row(uint32_t u) const {
    return rpb == 1 ? 0u : upr == 1 ? u : __umulhi(u, magic);  // 2^32 itself is no magic
  }
};

// upr is a multiple of 32 / V: a group never spans two rows, and the lanes of a group are
// inside the block's accesses together.
template <typename T, int V>
__global__ void __launch_bounds__(THREADS)
quantize_kernel(const T* x, int64_t ldx, const int64_t* ridx, int64_t src_rows, int64_t rows, int n, int8_t* codes,
                int64_t ldc, uint8_t* scales, int64_t lds, Units un, int* status) {
  const int64_t row0 = (int64_t)blockIdx.x * un.rpb;
  const uint32_t units = (uint32_t)mn<int64_t>(un.rpb, rows - row0) * (uint32_t)un.upr;
  for (uint32_t u0 = threadIdx.x; u0 - threadIdx.x < units; u0 += THREADS * UNROLL) {
    Raw<T, V> q[UNROLL];
    uint32_t lr[UNROLL];
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const uint32_t u = u0 + j * THREADS;
      lr[j] = un.row(u);
      memset(&q[j], 0, sizeof(q[j]));
      if (u < units) {
        const int64_t r = source_row(row0 + lr[j], ridx, src_rows, status);
        if (r >= 0) q[j] = load_raw<T, V>(x + r * ldx, (int)(u - lr[j] * un.upr) * V, n);
      }
    }
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const uint32_t u = u0 + j * THREADS;
      const int c = (int)(u - lr[j] * un.upr) * V;
      const int64_t i = row0 + lr[j];
      float v[V];
      unpack(q[j], v);
      const uint32_t m = q8::group_max_bits<V>(v), s = q8::scale_byte(m);
      if (u < units) {
        q8::store_codes<V>(codes + i * ldc + c, v, m, s);
        if ((c & (q8::GROUP - 1)) == 0) scales[i * lds + c / q8::GROUP] = (uint8_t)s;
      }
    }
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(THREADS)
dequantize_kernel(const int8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, const int64_t* ridx,
                  int64_t src_rows, int64_t rows, int n, T* out, int64_t ldo, Units un, int* status) {
  const int64_t row0 = (int64_t)blockIdx.x * un.rpb;
  const uint32_t units = (uint32_t)mn<int64_t>(un.rpb, rows - row0) * (uint32_t)un.upr;
  for (uint32_t u0 = threadIdx.x; u0 < units; u0 += THREADS * UNROLL) {
    q8::Codes<V> q[UNROLL];
    uint32_t lr[UNROLL], s[UNROLL];
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const uint32_t u = u0 + j * THREADS;
      lr[j] = un.row(u);
      q[j] = q8::Codes<V>{};
      s[j] = 0;
      if (u < units) {
        const int64_t r = source_row(row0 + lr[j], ridx, src_rows, status);
        const int c = (int)(u - lr[j] * un.upr) * V;
        if (r >= 0) {
          q[j] = q8::load_codes<V>(codes + r * ldc + c);
          s[j] = scales[r * lds + c / q8::GROUP];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const uint32_t u = u0 + j * THREADS;
      if (u >= units) continue;
      float v[V];
      q8::values<V>(q[j], q8::scale_of(s[j]), v);
      store_vec<V>(out + (row0 + lr[j]) * ldo, (int)(u - lr[j] * un.upr) * V, n, v);
    }
  }
}

// About 8 accesses a thread, fewer while the blocks would not fill the GPU twice.
Units units_of(int64_t rows, int64_t upr) {
  const int64_t want = std::clamp<int64_t>(rows * upr / (148 * 2), THREADS, 8 * THREADS);
  Units u;
  u.upr = (int)upr;
  u.rpb = (int)std::max<int64_t>(1, want / upr);
  u.magic = (uint32_t)(((1ull << 32) + upr - 1) / upr);
  return u;
}

template <typename T, int V>
void quantize(const void* x, int64_t ldx, const int64_t* ridx, int64_t src_rows, int64_t rows, int64_t n,
              int8_t* codes, int64_t ldc, uint8_t* scales, int64_t lds, int* status, cudaStream_t s) {
  const Units u = units_of(rows, q8::pitch(n) / V);
  quantize_kernel<T, V><<<(unsigned)cdiv(rows, u.rpb), THREADS, 0, s>>>((const T*)x, ldx, ridx, src_rows, rows, (int)n,
                                                                        codes, ldc, scales, lds, u, status);
}
template <typename T, int V>
void dequantize(const int8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, const int64_t* ridx,
                int64_t src_rows, int64_t rows, int64_t n, void* out, int64_t ldo, int* status, cudaStream_t s) {
  const Units u = units_of(rows, cdiv(n, V));
  dequantize_kernel<T, V><<<(unsigned)cdiv(rows, u.rpb), THREADS, 0, s>>>(codes, ldc, scales, lds, ridx, src_rows,
                                                                          rows, (int)n, (T*)out, ldo, u, status);
}

}  // namespace

int q8_quantize_run(const void* x, int64_t ldx, int dtype, const int64_t* ridx, int64_t src_rows, int64_t rows,
                    int64_t n, int8_t* codes, int64_t ldc, uint8_t* scales, int64_t lds, int* status,
                    cudaStream_t s) {
  using B = __nv_bfloat16;
  if (dtype == IFK_F32) {
    if (rows_allow<float>(x, ldx, 4))
      quantize<float, 4>(x, ldx, ridx, src_rows, rows, n, codes, ldc, scales, lds, status, s);
    else
      quantize<float, 1>(x, ldx, ridx, src_rows, rows, n, codes, ldc, scales, lds, status, s);
  } else if (rows_allow<B>(x, ldx, 8)) {
    quantize<B, 16>(x, ldx, ridx, src_rows, rows, n, codes, ldc, scales, lds, status, s);
  } else {
    quantize<B, 1>(x, ldx, ridx, src_rows, rows, n, codes, ldc, scales, lds, status, s);
  }
  IFK_CUDA_TRY(cudaGetLastError());
  return IFK_OK;
}

int q8_dequantize_run(const int8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, const int64_t* ridx,
                      int64_t src_rows, int64_t rows, int64_t n, void* out, int64_t ldo, int dtype, int* status,
                      cudaStream_t s) {
  using B = __nv_bfloat16;
  if (dtype == IFK_F32) {
    if (rows_allow<float>(out, ldo, 4))
      dequantize<float, 4>(codes, ldc, scales, lds, ridx, src_rows, rows, n, out, ldo, status, s);
    else
      dequantize<float, 1>(codes, ldc, scales, lds, ridx, src_rows, rows, n, out, ldo, status, s);
  } else if (rows_allow<B>(out, ldo, 8)) {
    dequantize<B, 8>(codes, ldc, scales, lds, ridx, src_rows, rows, n, out, ldo, status, s);
  } else {
    dequantize<B, 1>(codes, ldc, scales, lds, ridx, src_rows, rows, n, out, ldo, status, s);
  }
  IFK_CUDA_TRY(cudaGetLastError());
  return IFK_OK;
}

}  // namespace ifk
