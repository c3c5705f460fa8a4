// Layer norm, backward (ifk_layernorm_backward): dx, and the sums over the rows dw, db.
//
// Bound by memory: dy and the saved rows (as they were, or in 8 bits) are read once, dx
// is written once.  A team of W warps holds a row, 16 columns a lane; the teams of a
// persistent block walk the rows, each lane with the sums of its own 16 columns for dw
// and db in registers and the next row's loads in flight.  At the end the block adds its
// teams' sums in shared memory and writes one row of partial sums; a second kernel adds
// the blocks'.  The order of every sum is fixed by the sizes.
#include <algorithm>
#include <cstring>

#include "rowvec.cuh"
#include "ifk_internal.h"

namespace ifk {

namespace {

struct BwdArgs {
  const void* dy;
  const void* x;
  const int8_t* codes;
  const uint8_t* scales;
  const float* mean;
  const float* rstd;
  const void* w;
  void* dx;
  float* part;  // [2][blocks][n]: the blocks' sums of dy z and of dy; null: not wanted
  int64_t lddy, ldx, ldc, lds, lddx, rows;
  int n;
  bool w_bf16;
  int W, teams;  // warps a row, teams a block
};

constexpr int COLS = 16;       // columns a lane holds
constexpr int MAX_W = 16;      // warps a row: up to 32 * 16 * COLS = 8192 columns
constexpr int BLOCK_WARPS = 16;

// A barrier of one team's warps.
__device__ __forceinline__ void team_barrier(int team, int W) {
  asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(W * 32) : "memory");
}

// What a lane reads of a row.
template <typename TX, typename TY, int V, bool Q8, bool PLAIN>
struct RowIn {
  static constexpr int NV = COLS / V;
  Raw<TY, V> dy[NV];
  Raw<TX, V> x[Q8 ? 1 : NV];
  q8::Codes<V> c[Q8 ? NV : 1];
  uint8_t s[Q8 ? NV : 1];
  float mean, rstd;
  __device__ __forceinline__ void load(const BwdArgs& a, int64_t row, int c0, int step) {
    mean = a.mean[row];
    rstd = a.rstd[row];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int col = c0 + k * step;
      dy[k] = load_raw<TY, V, PLAIN>((const TY*)a.dy + row * a.lddy, col, a.n);
      if (Q8) {
        if (col < a.n) {
          c[k % (Q8 ? NV : 1)] = q8::load_codes<V>(a.codes + row * a.ldc + col);
          s[k % (Q8 ? NV : 1)] = a.scales[row * a.lds + col / q8::GROUP];
        } else {
          c[k % (Q8 ? NV : 1)] = q8::Codes<V>{};
          s[k % (Q8 ? NV : 1)] = 0;
        }
      } else {
        x[k % (Q8 ? 1 : NV)] = load_raw<TX, V, PLAIN>((const TX*)a.x + row * a.ldx, col, a.n);
      }
    }
  }
  // the saved values of access k
  __device__ __forceinline__ void saved(int k, float (&v)[V]) const {
    if (Q8) q8::values<V>(c[k % (Q8 ? NV : 1)], q8::scale_of(s[k % (Q8 ? NV : 1)]), v);
    else unpack(x[k % (Q8 ? 1 : NV)], v);
  }
};

// PLAIN: n is a multiple of V, w is there and fp32.
template <typename TX, typename TY, int V, bool Q8, bool PLAIN>
__global__ void __launch_bounds__(32 * BLOCK_WARPS, 1) backward_kernel(const BwdArgs a) {
  using In = RowIn<TX, TY, V, Q8, PLAIN>;
  constexpr int NV = In::NV;
  __shared__ float2 buf[2][BLOCK_WARPS];
  extern __shared__ float sums[];  // n, with several teams
  const int W = a.W, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int team = warp / W;
  const int c0 = ((warp - team * W) * 32 + lane) * V, step = 32 * W * V;
  const float inv_n = 1.f / (float)a.n;
  const int64_t stride = (int64_t)gridDim.x * a.teams;
  float sw[NV][V], sb[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) sw[k][i] = sb[k][i] = 0.f;
  int64_t row = (int64_t)blockIdx.x * a.teams + team;
  In in;
  if (row < a.rows) in.load(a, row, c0, step);
  for (int par = 0; row < a.rows; row += stride, par ^= 1) {
    // (one element an access, the unaligned case, has no registers left for a row ahead)
    In next;
    if (V > 1 && row + stride < a.rows) next.load(a, row + stride, c0, step);
    float g[NV][V], z[NV][V];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * step;
      unpack(in.dy[k], g[k]);
      if (PLAIN && c >= a.n) continue;  // dy is 0 there
      float w[V];
      if constexpr (PLAIN) load_f32<V>((const float*)a.w, c, w);
      else load_param<V>(a.w, a.w_bf16, 1.f, c, a.n, w);
      in.saved(k, z[k]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        z[k][i] = PLAIN || c + i < a.n ? (z[k][i] - in.mean) * in.rstd : 0.f;
        sw[k][i] = fmaf(g[k][i], z[k][i], sw[k][i]);
        sb[k][i] += g[k][i];
        g[k][i] = PLAIN || c + i < a.n ? g[k][i] * w[i] : 0.f;
        s.x += g[k][i];
        s.y = fmaf(g[k][i], z[k][i], s.y);
      }
    }
    s.x = warp_sum(s.x);
    s.y = warp_sum(s.y);
    if (W > 1) {
      // two buffers in turn: the barrier of the next row stands between its writes and these reads
      if (lane == 0) buf[par][warp] = s;
      team_barrier(team, W);
      s = make_float2(0.f, 0.f);
      for (int i = 0; i < W; ++i) {
        const float2 q = buf[par][team * W + i];
        s.x += q.x;
        s.y += q.y;
      }
    }
    const float m1 = s.x * inv_n * in.rstd, m2 = s.y * inv_n * in.rstd;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * step;
      if (c >= a.n) continue;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = fmaf(in.rstd, g[k][i], fmaf(-m2, z[k][i], -m1));
      store_vec<V, PLAIN>((TX*)a.dx + row * a.lddx, c, a.n, o);
    }
    if (V > 1) in = next;
    else if (row + stride < a.rows) in.load(a, row + stride, c0, step);
  }
  if (!a.part) return;
  for (int which = 0; which < 2; ++which) {
    float* out = a.part + ((int64_t)which * gridDim.x + blockIdx.x) * a.n;
    for (int q = 0; q < a.teams; ++q) {
      __syncthreads();
      if (q != team) continue;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int c = c0 + k * step + i;
          if (c >= a.n) continue;
          float v = which ? sb[k][i] : sw[k][i];
          if (q > 0) v += sums[c];
          if (q + 1 < a.teams) sums[c] = v;
          else out[c] = v;
        }
    }
  }
}

// Rows too wide for registers: dx by a block that walks its row twice ...
template <typename TX, typename TY, int V, bool Q8>
__device__ __forceinline__ void row_part(const BwdArgs& a, int64_t row, int c, float mean, float rstd, float (&g)[V],
                                         float (&z)[V]) {
  unpack(load_raw<TY, V>((const TY*)a.dy + row * a.lddy, c, a.n), g);
  if (Q8) {
    const q8::Codes<V> q = c < a.n ? q8::load_codes<V>(a.codes + row * a.ldc + c) : q8::Codes<V>{};
    q8::values<V>(q, c < a.n ? q8::scale_of(a.scales[row * a.lds + c / q8::GROUP]) : 0.f, z);
  } else {
    unpack(load_raw<TX, V>((const TX*)a.x + row * a.ldx, c, a.n), z);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) z[i] = c + i < a.n ? (z[i] - mean) * rstd : 0.f;
}

template <typename TX, typename TY, int V, bool Q8>
__global__ void __launch_bounds__(512) backward_long_kernel(const BwdArgs a) {
  __shared__ float2 buf[16];
  const int64_t row = blockIdx.x;
  const float mean = a.mean[row], rstd = a.rstd[row];
  float g[V], z[V], w[V];
  float2 s = make_float2(0.f, 0.f);
  for (int c = threadIdx.x * V; c < a.n; c += 512 * V) {
    row_part<TX, TY, V, Q8>(a, row, c, mean, rstd, g, z);
    load_param<V>(a.w, a.w_bf16, 1.f, c, a.n, w);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float gw = c + i < a.n ? g[i] * w[i] : 0.f;
      s.x += gw;
      s.y = fmaf(gw, z[i], s.y);
    }
  }
  s.x = warp_sum(s.x);
  s.y = warp_sum(s.y);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = s;
  __syncthreads();
  s = make_float2(0.f, 0.f);
  for (int i = 0; i < 16; ++i) {
    s.x += buf[i].x;
    s.y += buf[i].y;
  }
  const float inv_n = 1.f / (float)a.n, m1 = s.x * inv_n, m2 = s.y * inv_n;
  for (int c = threadIdx.x * V; c < a.n; c += 512 * V) {
    row_part<TX, TY, V, Q8>(a, row, c, mean, rstd, g, z);
    load_param<V>(a.w, a.w_bf16, 1.f, c, a.n, w);
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = rstd * (g[i] * w[i] - m1 - z[i] * m2);
    store_vec<V>((TX*)a.dx + row * a.lddx, c, a.n, o);
  }
}

// ... and dw, db by blocks of 32 V columns that walk a share of the rows, each warp every
// eighth of them; the warps' sums are added in order.
template <typename TX, typename TY, int V, bool Q8>
__global__ void __launch_bounds__(256) backward_long_sums_kernel(const BwdArgs a) {
  __shared__ float sum[2][32 * V];
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 * V + lane * V;
  float sw[V], sb[V];
#pragma unroll
  for (int i = 0; i < V; ++i) sw[i] = sb[i] = 0.f;
  for (int64_t row = (int64_t)blockIdx.y * 8 + wp; row < a.rows; row += (int64_t)gridDim.y * 8) {
    float g[V], z[V];
    row_part<TX, TY, V, Q8>(a, row, c, a.mean[row], a.rstd[row], g, z);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      sw[i] = fmaf(g[i], z[i], sw[i]);
      sb[i] += g[i];
    }
  }
  for (int q = 0; q < 8; ++q) {
    __syncthreads();
    if (q != wp) continue;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      sum[0][lane * V + i] = q == 0 ? sw[i] : sum[0][lane * V + i] + sw[i];
      sum[1][lane * V + i] = q == 0 ? sb[i] : sum[1][lane * V + i] + sb[i];
    }
  }
  __syncthreads();
  const int k = threadIdx.x;
  const int cc = blockIdx.x * 32 * V + k;
  if (k < 32 * V && cc < a.n) {
    a.part[(int64_t)blockIdx.y * a.n + cc] = sum[0][k];
    a.part[((int64_t)gridDim.y + blockIdx.y) * a.n + cc] = sum[1][k];
  }
}

// Persistent blocks: one an SM, fewer when the rows do not fill them (the partial sums are
// written and read once a block).
int row_warps(int64_t n) { return (int)cdiv(n, 32 * COLS); }
int block_teams(int64_t n) { return std::max(1, BLOCK_WARPS / row_warps(n)); }
int64_t parts_of(int64_t rows, int64_t n) {
  if (row_warps(n) > MAX_W) return std::min<int64_t>(cdiv(rows, 64), 32);
  return std::min<int64_t>(cdiv(rows, block_teams(n)), 148);
}

template <typename TX, typename TY, int V, bool Q8>
int backward(BwdArgs& a, cudaStream_t s) {
  const int64_t parts = parts_of(a.rows, a.n);
  a.W = row_warps(a.n);
  if (a.W > MAX_W) {
    backward_long_kernel<TX, TY, V, Q8><<<(unsigned)a.rows, 512, 0, s>>>(a);
    if (a.part)
      backward_long_sums_kernel<TX, TY, V, Q8>
          <<<dim3((unsigned)cdiv(a.n, 32 * V), (unsigned)parts), 256, 0, s>>>(a);
  } else {
    a.teams = block_teams(a.n);
    const size_t smem = a.part && a.teams > 1 ? (size_t)a.n * sizeof(float) : 0;
    const unsigned threads = 32 * a.W * a.teams;
    if (V > 1 && a.n % V == 0 && a.w && !a.w_bf16)
      backward_kernel<TX, TY, V, Q8, V != 1><<<(unsigned)parts, threads, smem, s>>>(a);
    else
      backward_kernel<TX, TY, V, Q8, false><<<(unsigned)parts, threads, smem, s>>>(a);
  }
  IFK_CUDA_TRY(cudaGetLastError());
  return IFK_OK;
}

template <typename TX, typename TY>
int backward_any(BwdArgs& a, cudaStream_t s) {
  constexpr int V = sizeof(TX) == 2 && sizeof(TY) == 2 ? 8 : 4;
  const bool al = rows_allow<TY>(a.dy, a.lddy, V) && rows_allow<TX>(a.dx, a.lddx, V) &&
                  (!a.x || rows_allow<TX>(a.x, a.ldx, V)) && ((uintptr_t)a.w & 15) == 0;
  if (a.x) return al ? backward<TX, TY, V, false>(a, s) : backward<TX, TY, 1, false>(a, s);
  return al ? backward<TX, TY, V, true>(a, s) : backward<TX, TY, 1, true>(a, s);
}

// out[c] = sum over p of part[p][c] in a fixed order: 32 threads a column take every
// 32nd p, then one adds the 32.
__global__ void __launch_bounds__(1024) sum_parts_kernel(const float* part, int64_t parts, int64_t n, float* out,
                                                         const float* part2, float* out2, int accumulate) {
  __shared__ float sh[32][33];
  const float* src = blockIdx.y ? part2 : part;
  float* dst = blockIdx.y ? out2 : out;
  if (!dst) return;
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  if (c < n)
    for (int64_t p = threadIdx.y; p < parts; p += 32) v += src[p * n + c];
  sh[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  // the 32 sums of a column, one to a lane
  v = warp_sum(sh[threadIdx.x][threadIdx.y]);
  const int64_t o = (int64_t)blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && o < n) dst[o] = accumulate ? dst[o] + v : v;
}

}  // namespace

int sum_parts_run(const float* part, int64_t parts, int64_t n, float* out, const float* part2, float* out2,
                  int accumulate, cudaStream_t s) {
  const dim3 grid((unsigned)cdiv(n, 32), part2 ? 2 : 1);
  sum_parts_kernel<<<grid, dim3(32, 32), 0, s>>>(part, parts, n, out, part2, out2, accumulate);
  IFK_CUDA_TRY(cudaGetLastError());
  return IFK_OK;
}

size_t layernorm_backward_bytes(int64_t rows, int64_t n) {
  return (size_t)std::max<int64_t>(parts_of(rows, n), 1) * (size_t)n * 2 * sizeof(float);
}

int layernorm_backward_run(const void* dy, int64_t lddy, int y_dtype, const void* x, int64_t ldx, int x_dtype,
                           const int8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, const float* mean,
                           const float* rstd, const void* w, int w_dtype, int64_t rows, int64_t n, void* dx,
                           int64_t lddx, float* dw, float* db, float* part, cudaStream_t s) {
  BwdArgs a;
  a.dy = dy;
  a.x = x;
  a.codes = codes;
  a.scales = scales;
  a.mean = mean;
  a.rstd = rstd;
  a.w = w;
  a.dx = dx;
  a.part = (dw || db) ? part : nullptr;
  a.lddy = lddy;
  a.ldx = ldx;
  a.ldc = ldc;
  a.lds = lds;
  a.lddx = lddx;
  a.rows = rows;
  a.n = (int)n;
  a.w_bf16 = w_dtype == IFK_BF16;
  a.teams = 1;
  using B = __nv_bfloat16;
  int rc;
  if (x_dtype == IFK_F32) rc = y_dtype == IFK_F32 ? backward_any<float, float>(a, s) : backward_any<float, B>(a, s);
  else rc = y_dtype == IFK_F32 ? backward_any<B, float>(a, s) : backward_any<B, B>(a, s);
  if (rc != IFK_OK || !a.part) return rc;
  const int64_t parts = parts_of(rows, n);
  return sum_parts_run(part, parts, n, dw, part + parts * n, db, 0, s);
}

}  // namespace ifk
