// Activation rows to 8 bits and back (ifk_q8_quantize, ifk_q8_dequantize).
//
// Both are one pass bound by memory: 2 (bf16) or 4 (fp32) bytes an element on one
// side, 1 + 1/32 on the other.  A thread takes 8 neighbouring columns (one or two
// 16-byte accesses of the rows, 8 bytes of codes), four neighbouring lanes a
// group, so the group's maximum is two shuffles and no shared memory is needed.
#include "q8.cuh"
#include "ifk_internal.h"

namespace ifk {

namespace {

constexpr int THREADS = 256;

// Row i of a call: the row itself, or its entry in the index (-1: out of range).
__device__ __forceinline__ int64_t source_row(int64_t i, const int64_t* ridx, int64_t src_rows, int* status) {
  if (!ridx) return i;
  const int64_t r = ridx[i];
  if (r >= 0 && r < src_rows) return r;
  if (status) *status = IFK_ERR_ARG;
  return -1;
}

// A block takes `rpb` whole rows: unit u of the block is 8 columns of row u / upr.
// upr is a multiple of 4, so the quad of a group never spans two rows, and the
// tail threads of a block stay in the loop for the shuffles.
template <typename T>
__global__ void __launch_bounds__(THREADS)
quantize_kernel(const T* x, int64_t ldx, bool vec, const int64_t* ridx, int64_t src_rows, int64_t rows, int64_t n,
                int8_t* codes, int64_t ldc, uint8_t* scales, int64_t lds, int upr, int rpb, int* status) {
  const int64_t row0 = (int64_t)blockIdx.x * rpb;
  const uint32_t units = (uint32_t)(mn<int64_t>(rpb, rows - row0)) * (uint32_t)upr;
  for (uint32_t u0 = 0; u0 < units; u0 += THREADS) {
    const uint32_t u = u0 + threadIdx.x;
    const bool on = u < units;
    const uint32_t lr = on ? u / (uint32_t)upr : 0;
    const int64_t i = row0 + lr, c = (int64_t)(u - lr * (uint32_t)upr) * q8::VEC;
    float v[q8::VEC] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (on) {
      const int64_t r = source_row(i, ridx, src_rows, status);
      if (r >= 0) load8(x + r * ldx, c, n, vec, v);
    }
    const uint32_t s = q8::scale_byte(q8::group_max(v));
    if (on) {
      *reinterpret_cast<uint2*>(codes + i * ldc + c) = q8::codes8(v, s);
      if ((threadIdx.x & 3) == 0) scales[i * lds + c / q8::GROUP] = (uint8_t)s;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
dequantize_kernel(const int8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, const int64_t* ridx,
                  int64_t src_rows, int64_t rows, int64_t n, T* out, int64_t ldo, bool vec, int upr, int rpb,
                  int* status) {
  const int64_t row0 = (int64_t)blockIdx.x * rpb;
  const uint32_t units = (uint32_t)(mn<int64_t>(rpb, rows - row0)) * (uint32_t)upr;
  for (uint32_t u = threadIdx.x; u < units; u += THREADS) {
    const uint32_t lr = u / (uint32_t)upr;
    const int64_t i = row0 + lr, c = (int64_t)(u - lr * (uint32_t)upr) * q8::VEC;
    const int64_t r = source_row(i, ridx, src_rows, status);
    float v[q8::VEC] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (r >= 0)
      q8::values8(*reinterpret_cast<const uint2*>(codes + r * ldc + c),
                  q8::scale_of(scales[r * lds + c / q8::GROUP]), v);
    store8(out + i * ldo, c, n, vec, v);
  }
}

// Rows a block takes: about 8 units a thread, whole rows.
int rows_per_block(int upr) { return (int)mx<int64_t>(1, cdiv(8 * THREADS, upr)); }

}  // namespace

int q8_quantize_run(const void* x, int64_t ldx, int dtype, const int64_t* ridx, int64_t src_rows, int64_t rows,
                    int64_t n, int8_t* codes, int64_t ldc, uint8_t* scales, int64_t lds, int* status,
                    cudaStream_t s) {
  const int upr = (int)(q8::pitch(n) / q8::VEC), rpb = rows_per_block(upr);
  const unsigned grid = (unsigned)cdiv(rows, rpb);
  if (dtype == IFK_F32)
    quantize_kernel<float><<<grid, THREADS, 0, s>>>((const float*)x, ldx, rows_aligned((const float*)x, ldx), ridx,
                                                    src_rows, rows, n, codes, ldc, scales, lds, upr, rpb, status);
  else
    quantize_kernel<__nv_bfloat16><<<grid, THREADS, 0, s>>>(
        (const __nv_bfloat16*)x, ldx, rows_aligned((const __nv_bfloat16*)x, ldx), ridx, src_rows, rows, n, codes, ldc,
        scales, lds, upr, rpb, status);
  IFK_CUDA_TRY(cudaGetLastError());
  return IFK_OK;
}

int q8_dequantize_run(const int8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, const int64_t* ridx,
                      int64_t src_rows, int64_t rows, int64_t n, void* out, int64_t ldo, int dtype, int* status,
                      cudaStream_t s) {
  const int upr = (int)(cdiv(n, q8::VEC)), rpb = rows_per_block(upr);
  const unsigned grid = (unsigned)cdiv(rows, rpb);
  if (dtype == IFK_F32)
    dequantize_kernel<float><<<grid, THREADS, 0, s>>>(codes, ldc, scales, lds, ridx, src_rows, rows, n, (float*)out,
                                                      ldo, rows_aligned((float*)out, ldo), upr, rpb, status);
  else
    dequantize_kernel<__nv_bfloat16><<<grid, THREADS, 0, s>>>(codes, ldc, scales, lds, ridx, src_rows, rows, n,
                                                              (__nv_bfloat16*)out, ldo,
                                                              rows_aligned((__nv_bfloat16*)out, ldo), upr, rpb,
                                                              status);
  IFK_CUDA_TRY(cudaGetLastError());
  return IFK_OK;
}

}  // namespace ifk
