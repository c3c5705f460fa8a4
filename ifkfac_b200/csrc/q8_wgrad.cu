// Weight and bias gradient of a linear layer from its 8-bit input rows
// (ifk_q8_wgrad): dW = delta^T X, db = column sums of delta.
#include "q8.cuh"
#include "ifk_internal.h"

namespace ifk {

namespace {

constexpr int TILE = 64, KB = 16;

// 64 x 64 of dW by 256 threads, 4 x 4 each, 16 rows at a time through shared memory.
template <typename TD>
__global__ void __launch_bounds__(256)
wgrad_kernel(const TD* delta, int64_t ldd, const int8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds,
             int64_t rows, int64_t n_out, int64_t n_in, float* dW, int64_t ldw, int accumulate) {
  __shared__ float sd[KB][TILE + 4], sx[KB][TILE + 4];
  const int64_t i0 = (int64_t)blockIdx.x * TILE, o0 = (int64_t)blockIdx.y * TILE;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int64_t r0 = 0; r0 < rows; r0 += KB) {
    for (int u = threadIdx.x; u < KB * TILE; u += 256) {
      const int k = u / TILE, c = u % TILE;
      const int64_t r = r0 + k;
      sd[k][c] = r < rows && o0 + c < n_out ? ld_elem(delta, r * ldd + o0 + c) : 0.f;
      float x = 0.f;
      if (r < rows && i0 + c < n_in)
        x = (float)codes[r * ldc + i0 + c] * q8::scale_of(scales[r * lds + (i0 + c) / q8::GROUP]);
      sx[k][c] = x;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[p][q] = fmaf(sd[k][ty * 4 + p], sx[k][tx * 4 + q], acc[p][q]);
    __syncthreads();
  }
  for (int p = 0; p < 4; ++p)
    for (int q = 0; q < 4; ++q) {
      const int64_t o = o0 + ty * 4 + p, i = i0 + tx * 4 + q;
      if (o < n_out && i < n_in) {
        float* d = dW + o * ldw + i;
        *d = accumulate ? *d + acc[p][q] : acc[p][q];
      }
    }
}

// Sums over a share of the rows of 256 columns, 8 a lane; warps take every eighth row
// of the share and are added in order.
template <typename TD>
__global__ void __launch_bounds__(256)
column_sums_kernel(const TD* d, int64_t ldd, bool vec, int64_t rows, int64_t n, float* part) {
  __shared__ float sum[256];
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 256 + lane * 8;
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int64_t r = (int64_t)blockIdx.y * 8 + wp; r < rows; r += (int64_t)gridDim.y * 8) {
    float v[8];
    load8(d + r * ldd, c, n, vec, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] += v[i];
  }
  for (int q = 0; q < 8; ++q) {
    __syncthreads();
    if (q != wp) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[lane * 8 + i] = q == 0 ? s[i] : sum[lane * 8 + i] + s[i];
  }
  __syncthreads();
  const int64_t cc = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (cc < n) part[(int64_t)blockIdx.y * n + cc] = sum[threadIdx.x];
}

int64_t sum_splits(int64_t rows, int64_t n) {
  return mx<int64_t>(1, mn<int64_t>(cdiv(rows, 64), 148 * 4 / cdiv(n, 256)));
}

template <typename TD>
int run(const TD* delta, int64_t ldd, const int8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds,
        int64_t rows, int64_t n_out, int64_t n_in, float* dW, int64_t ldw, float* db, int accumulate, uint8_t* ws,
        cudaStream_t s) {
  const dim3 grid((unsigned)cdiv(n_in, TILE), (unsigned)cdiv(n_out, TILE));
  wgrad_kernel<TD><<<grid, 256, 0, s>>>(delta, ldd, codes, ldc, scales, lds, rows, n_out, n_in, dW, ldw, accumulate);
  IFK_CUDA_TRY(cudaGetLastError());
  if (!db) return IFK_OK;
  const int64_t parts = sum_splits(rows, n_out);
  column_sums_kernel<TD><<<dim3((unsigned)cdiv(n_out, 256), (unsigned)parts), 256, 0, s>>>(
      delta, ldd, rows_aligned(delta, ldd), rows, n_out, (float*)ws);
  IFK_CUDA_TRY(cudaGetLastError());
  return sum_parts_run((float*)ws, parts, n_out, db, nullptr, nullptr, accumulate, s);
}

}  // namespace

size_t q8_wgrad_bytes(int64_t rows, int64_t n_out, int64_t n_in, int dtype) {
  (void)n_in;
  (void)dtype;
  return (size_t)sum_splits(rows, n_out) * (size_t)n_out * sizeof(float);
}

int q8_wgrad_run(const void* delta, int64_t ldd, int dtype, const int8_t* codes, int64_t ldc, const uint8_t* scales,
                 int64_t lds, int64_t rows, int64_t n_out, int64_t n_in, float* dW, int64_t ldw, float* db,
                 int accumulate, int* status, uint8_t* ws, cudaStream_t s) {
  (void)status;
  if (dtype == IFK_F32)
    return run((const float*)delta, ldd, codes, ldc, scales, lds, rows, n_out, n_in, dW, ldw, db, accumulate, ws, s);
  return run((const __nv_bfloat16*)delta, ldd, codes, ldc, scales, lds, rows, n_out, n_in, dW, ldw, db, accumulate,
             ws, s);
}

}  // namespace ifk
