// extern "C" entry points of the 8-bit activation rows and the layer norm
// (declared in include/ifk.h).  Host-side validation happens before anything is queued.
#include <cmath>

#include "q8.cuh"
#include "ifk_internal.h"

using namespace ifk;

namespace {

constexpr size_t ALIGN = 256;
size_t align_up(size_t b) { return (b + ALIGN - 1) / ALIGN * ALIGN; }
bool aligned(const void* p) { return ((uintptr_t)p % ALIGN) == 0; }
bool dtype_ok(int d) { return d == IFK_F32 || d == IFK_BF16; }
cudaStream_t S(ifk_stream_t s) { return (cudaStream_t)s; }

// Largest width, and largest side of a weight gradient: columns and tiles are 32-bit in the kernels.
constexpr int64_t MAX_SIDE = 1 << 28;

// Layout of 8-bit rows of n columns.
int q8_rows_ok(const int8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, int64_t n) {
  if (!codes || !scales || ((uintptr_t)codes & 15)) return IFK_ERR_ARG;
  if (ldc < q8::pitch(n) || ldc % 16 != 0 || lds < q8::pitch(n) / q8::GROUP) return IFK_ERR_SHAPE;
  return IFK_OK;
}

}  // namespace

extern "C" {

int64_t ifk_q8_pitch(int64_t n) { return n <= 0 ? 0 : q8::pitch(n); }

int ifk_q8_quantize(const void* x, int64_t ld_x, int dtype, const int64_t* row_index, int64_t src_rows, int64_t rows,
                    int64_t n, int8_t* codes, int64_t ld_codes, uint8_t* scales, int64_t ld_scales, int* d_status,
                    ifk_stream_t stream) {
  if (rows < 0 || n <= 0 || n > MAX_SIDE) return IFK_ERR_SHAPE;
  if (!dtype_ok(dtype)) return IFK_ERR_DTYPE;
  if (rows == 0) return IFK_OK;
  if (!x) return IFK_ERR_ARG;
  if (ld_x < n || (row_index && src_rows <= 0)) return IFK_ERR_SHAPE;
  const int rc = q8_rows_ok(codes, ld_codes, scales, ld_scales, n);
  if (rc != IFK_OK) return rc;
  return q8_quantize_run(x, ld_x, dtype, row_index, src_rows, rows, n, codes, ld_codes, scales, ld_scales, d_status,
                         S(stream));
}

int ifk_q8_dequantize(const int8_t* codes, int64_t ld_codes, const uint8_t* scales, int64_t ld_scales,
                      const int64_t* row_index, int64_t src_rows, int64_t rows, int64_t n, void* out, int64_t ld_out,
                      int out_dtype, int* d_status, ifk_stream_t stream) {
  if (rows < 0 || n <= 0 || n > MAX_SIDE) return IFK_ERR_SHAPE;
  if (!dtype_ok(out_dtype)) return IFK_ERR_DTYPE;
  if (rows == 0) return IFK_OK;
  if (!out) return IFK_ERR_ARG;
  if (ld_out < n || (row_index && src_rows <= 0)) return IFK_ERR_SHAPE;
  const int rc = q8_rows_ok(codes, ld_codes, scales, ld_scales, n);
  if (rc != IFK_OK) return rc;
  return q8_dequantize_run(codes, ld_codes, scales, ld_scales, row_index, src_rows, rows, n, out, ld_out, out_dtype,
                           d_status, S(stream));
}

size_t ifk_q8_wgrad_workspace(int64_t rows, int64_t n_out, int64_t n_in, int delta_dtype) {
  const bool in_place = delta_dtype == (IFK_BF16 | IFK_DELTA_IN_PLACE);
  if (in_place) delta_dtype = IFK_BF16;
  if (rows < 0 || n_out <= 0 || n_in <= 0 || !dtype_ok(delta_dtype)) return 0;
  if (rows > MAX_SIDE || n_out > MAX_SIDE || n_in > MAX_SIDE) return 0;
  return align_up(q8_wgrad_bytes(rows, n_out, n_in, delta_dtype, !in_place)) + ALIGN;
}

int ifk_q8_wgrad(const void* delta, int64_t ld_delta, int delta_dtype, const int8_t* codes, int64_t ld_codes,
                 const uint8_t* scales, int64_t ld_scales, int64_t rows, int64_t n_out, int64_t n_in, float* dW,
                 int64_t ld_dW, float* db, int accumulate, int* d_status, void* workspace, size_t workspace_bytes,
                 ifk_stream_t stream) {
  const bool withhold = delta_dtype & IFK_DEBUG_WITHHOLD;
  delta_dtype &= ~IFK_DEBUG_WITHHOLD;
  const int sized_as = delta_dtype;
  const bool in_place = delta_dtype == (IFK_BF16 | IFK_DELTA_IN_PLACE);
  if (in_place) delta_dtype = IFK_BF16;
  if (!dW) return IFK_ERR_ARG;
  if (rows < 0 || n_out <= 0 || n_in <= 0 || ld_dW < n_in) return IFK_ERR_SHAPE;
  if (rows > MAX_SIDE || n_out > MAX_SIDE || n_in > MAX_SIDE) return IFK_ERR_SHAPE;
  if (!dtype_ok(delta_dtype)) return IFK_ERR_DTYPE;
  cudaStream_t s = S(stream);
  if (rows == 0) {
    if (accumulate) return IFK_OK;
    IFK_CUDA_TRY(cudaMemset2DAsync(dW, (size_t)ld_dW * sizeof(float), 0, (size_t)n_in * sizeof(float), (size_t)n_out,
                                   s));
    if (db) IFK_CUDA_TRY(cudaMemsetAsync(db, 0, (size_t)n_out * sizeof(float), s));
    return IFK_OK;
  }
  if (!delta) return IFK_ERR_ARG;
  if (ld_delta < n_out) return IFK_ERR_SHAPE;
  if (in_place && (((uintptr_t)delta & 15) || ld_delta % 8)) return IFK_ERR_ARG;
  const int rc = q8_rows_ok(codes, ld_codes, scales, ld_scales, n_in);
  if (rc != IFK_OK) return rc;
  if (!workspace || !aligned(workspace) ||
      workspace_bytes < ifk_q8_wgrad_workspace(rows, n_out, n_in, sized_as))
    return IFK_ERR_WORKSPACE;
  return q8_wgrad_run(delta, ld_delta, delta_dtype, codes, ld_codes, scales, ld_scales, rows, n_out, n_in, dW, ld_dW,
                      db, accumulate ? 1 : 0, d_status, (uint8_t*)workspace, withhold, s);
}

int ifk_layernorm(const void* x, int64_t ld_x, int x_dtype, const void* w, const void* b, int w_dtype, int64_t rows,
                  int64_t n, double eps, void* y, int64_t ld_y, int y_dtype, float* mean, float* rstd, int8_t* codes,
                  int64_t ld_codes, uint8_t* scales, int64_t ld_scales, ifk_stream_t stream) {
  if (rows < 0 || n <= 0 || n > MAX_SIDE) return IFK_ERR_SHAPE;
  if (!dtype_ok(x_dtype) || !dtype_ok(y_dtype) || ((w || b) && !dtype_ok(w_dtype))) return IFK_ERR_DTYPE;
  if (!(eps >= 0) || std::isinf(eps)) return IFK_ERR_ARG;
  if (rows == 0) return IFK_OK;
  if (!x || !y || (codes == nullptr) != (scales == nullptr)) return IFK_ERR_ARG;
  if (ld_x < n || ld_y < n) return IFK_ERR_SHAPE;
  if (codes) {
    const int rc = q8_rows_ok(codes, ld_codes, scales, ld_scales, n);
    if (rc != IFK_OK) return rc;
  }
  return layernorm_run(x, ld_x, x_dtype, w, b, w_dtype, rows, n, eps, y, ld_y, y_dtype, mean, rstd, codes, ld_codes,
                       scales, ld_scales, S(stream));
}

size_t ifk_layernorm_backward_workspace(int64_t rows, int64_t n) {
  if (rows < 0 || n <= 0 || n > MAX_SIDE) return 0;
  return align_up(layernorm_backward_bytes(rows, n));
}

int ifk_layernorm_backward(const void* dy, int64_t ld_dy, int y_dtype, const void* x, int64_t ld_x, int x_dtype,
                           const int8_t* codes, int64_t ld_codes, const uint8_t* scales, int64_t ld_scales,
                           const float* mean, const float* rstd, const void* w, int w_dtype, int64_t rows, int64_t n,
                           void* dx, int64_t ld_dx, float* dw, float* db, int* d_status, void* workspace,
                           size_t workspace_bytes, ifk_stream_t stream) {
  const bool withhold = y_dtype & IFK_DEBUG_WITHHOLD;
  y_dtype &= ~IFK_DEBUG_WITHHOLD;
  if (rows < 0 || n <= 0 || n > MAX_SIDE) return IFK_ERR_SHAPE;
  if (!dtype_ok(x_dtype) || !dtype_ok(y_dtype) || (w && !dtype_ok(w_dtype))) return IFK_ERR_DTYPE;
  cudaStream_t s = S(stream);
  if (rows == 0) {
    if (dw) IFK_CUDA_TRY(cudaMemsetAsync(dw, 0, (size_t)n * sizeof(float), s));
    if (db) IFK_CUDA_TRY(cudaMemsetAsync(db, 0, (size_t)n * sizeof(float), s));
    return IFK_OK;
  }
  if (!dy || !mean || !rstd || !dx) return IFK_ERR_ARG;
  if ((x != nullptr) == (codes != nullptr)) return IFK_ERR_ARG;  // the saved rows in exactly one form
  if (ld_dy < n || ld_dx < n || (x && ld_x < n)) return IFK_ERR_SHAPE;
  if (codes) {
    const int rc = q8_rows_ok(codes, ld_codes, scales, ld_scales, n);
    if (rc != IFK_OK) return rc;
  }
  if ((dw || db) && (!workspace || !aligned(workspace) ||
                     workspace_bytes < ifk_layernorm_backward_workspace(rows, n)))
    return IFK_ERR_WORKSPACE;
  return layernorm_backward_run(dy, ld_dy, y_dtype, x, ld_x, x_dtype, codes, ld_codes, scales, ld_scales, mean, rstd,
                                w, w_dtype, rows, n, dx, ld_dx, dw, db, (float*)workspace, d_status, withhold, s);
}

}  // extern "C"
