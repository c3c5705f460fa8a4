// Layer norm forward and backward (ifk_layernorm, ifk_layernorm_backward).
//
// Bound by memory: the forward pass reads x and writes y (and the 8-bit rows of x
// when asked), the backward pass reads dy and the saved rows and writes dx; the
// sums over rows for dw and db stay in registers while a block walks its rows.
//
// A row is held in registers by a team of threads, 8 neighbouring columns
// ("a chunk") at a time: thread t of the team holds chunks t, t + TEAM, ...
#include "q8.cuh"
#include "ifk_internal.h"

namespace ifk {

namespace {

template <typename TW>
struct Affine {
  const TW* w;
  const TW* b;
};

// Sum over the TEAM threads of a row (a warp, or the whole block).  buf: 2 x 32 floats
// used in turn, so that one barrier a sum is enough.
template <int TEAM>
__device__ __forceinline__ float team_sum(float v, float* buf) {
  v = warp_sum(v);
  if (TEAM == 32) return v;
  const int w = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) buf[w] = v;
  __syncthreads();
  float r = 0.f;
#pragma unroll
  for (int i = 0; i < TEAM / 32; ++i) r += buf[i];
  return r;
}
template <int TEAM>
__device__ __forceinline__ float2 team_sum2(float2 v, float2* buf) {
  v.x = warp_sum(v.x);
  v.y = warp_sum(v.y);
  if (TEAM == 32) return v;
  const int w = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) buf[w] = v;
  __syncthreads();
  float2 r = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < TEAM / 32; ++i) {
    r.x += buf[i].x;
    r.y += buf[i].y;
  }
  return r;
}

struct FwdArgs {
  const void* x;
  const void* w;
  const void* b;
  void* y;
  float* mean;
  float* rstd;
  int8_t* codes;
  uint8_t* scales;
  int64_t ldx, ldy, ldc, lds, rows, n;
  float eps;
  bool vx, vy, vw;  // 16-byte accesses of x, y, and w with b
};

template <typename TW>
__device__ __forceinline__ void affine8(const void* w, const void* b, int64_t c, int64_t n, bool vec, float (&wv)[8],
                                        float (&bv)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    wv[i] = 1.f;
    bv[i] = 0.f;
  }
  if (w) load8((const TW*)w, c, n, vec, wv);
  if (b) load8((const TW*)b, c, n, vec, bv);
}

// 8 columns of the 8-bit rows of x, written as ifk_q8_quantize writes them.
__device__ __forceinline__ void write_codes(const FwdArgs& a, int64_t row, int64_t c, const float (&v)[8], bool on) {
  const uint32_t s = q8::scale_byte(q8::group_max(v));
  if (!on) return;
  *reinterpret_cast<uint2*>(a.codes + row * a.ldc + c) = q8::codes8(v, s);
  if ((threadIdx.x & 3) == 0) a.scales[row * a.lds + c / q8::GROUP] = (uint8_t)s;
}

// One row a team, rows up to TEAM * NCH * 8 columns.  The mean is taken twice:
// the second sum, over x less the first mean, carries what the first one rounded
// away, and the variance is that of the differences.
template <typename TX, typename TY, typename TW, int TEAM, int NCH, int BLOCK>
__global__ void __launch_bounds__(BLOCK) forward_kernel(FwdArgs a) {
  __shared__ float buf[2][32];
  const int t = TEAM == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const int64_t row = TEAM == 32 ? (int64_t)blockIdx.x * (BLOCK / 32) + (threadIdx.x >> 5) : blockIdx.x;
  if (TEAM == 32 && row >= a.rows) return;  // whole warps
  const TX* x = (const TX*)a.x + row * a.ldx;
  const float inv_n = 1.f / (float)a.n;
  float v[NCH][8];
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    load8(x, (int64_t)(t + k * TEAM) * 8, a.n, a.vx, v[k]);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += v[k][i];
  }
  const float m1 = team_sum<TEAM>(s, buf[0]) * inv_n;
  float2 d = make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    const int64_t c = (int64_t)(t + k * TEAM) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = c + i < a.n ? v[k][i] - m1 : 0.f;
      d.x += e;
      d.y = fmaf(e, e, d.y);
    }
  }
  __shared__ float2 buf2[32];
  d = team_sum2<TEAM>(d, buf2);
  const float c1 = d.x * inv_n;
  const float var = fmaxf(fmaf(-c1, c1, d.y * inv_n), 0.f);
  const float mean = m1 + c1, rstd = 1.f / sqrtf(var + a.eps);
  if (t == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
  TY* y = (TY*)a.y + row * a.ldy;
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    const int64_t c = (int64_t)(t + k * TEAM) * 8;
    if (a.codes) write_codes(a, row, c, v[k], c < a.ldc && c < cdiv(a.n, q8::GROUP) * q8::GROUP);
    if (c >= a.n) continue;
    float w[8], b[8], o[8];
    affine8<TW>(a.w, a.b, c, a.n, a.vw, w, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = fmaf((v[k][i] - m1 - c1) * rstd, w[i], b[i]);
    store8(y, c, a.n, a.vy, o);
  }
}

// Any width: a block walks its row three times.
template <typename TX, typename TY, typename TW, int BLOCK>
__global__ void __launch_bounds__(BLOCK) forward_long_kernel(FwdArgs a) {
  __shared__ float buf[32];
  __shared__ float2 buf2[32];
  const int64_t row = blockIdx.x;
  const TX* x = (const TX*)a.x + row * a.ldx;
  TY* y = (TY*)a.y + row * a.ldy;
  const int64_t pitch = q8::pitch(a.n);
  const float inv_n = 1.f / (float)a.n;
  float v[8], s = 0.f;
  for (int64_t c = (int64_t)threadIdx.x * 8; c < a.n; c += BLOCK * 8) {
    load8(x, c, a.n, a.vx, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += v[i];
  }
  const float m1 = team_sum<BLOCK>(s, buf) * inv_n;
  float2 d = make_float2(0.f, 0.f);
  for (int64_t c = (int64_t)threadIdx.x * 8; c < a.n; c += BLOCK * 8) {
    load8(x, c, a.n, a.vx, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = c + i < a.n ? v[i] - m1 : 0.f;
      d.x += e;
      d.y = fmaf(e, e, d.y);
    }
  }
  d = team_sum2<BLOCK>(d, buf2);
  const float c1 = d.x * inv_n;
  const float var = fmaxf(fmaf(-c1, c1, d.y * inv_n), 0.f);
  const float mean = m1 + c1, rstd = 1.f / sqrtf(var + a.eps);
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[row] = mean;
    if (a.rstd) a.rstd[row] = rstd;
  }
  // the loop bound is the same for the whole block: the groups' shuffles need every lane
  for (int64_t c0 = 0; c0 < pitch; c0 += BLOCK * 8) {
    const int64_t c = c0 + (int64_t)threadIdx.x * 8;
    load8(x, c, a.n, a.vx, v);
    if (a.codes) write_codes(a, row, c, v, c < pitch);
    if (c >= a.n) continue;
    float w[8], b[8], o[8];
    affine8<TW>(a.w, a.b, c, a.n, a.vw, w, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = fmaf((v[i] - m1 - c1) * rstd, w[i], b[i]);
    store8(y, c, a.n, a.vy, o);
  }
}

struct BwdArgs {
  const void* dy;
  const void* x;
  const int8_t* codes;
  const uint8_t* scales;
  const float* mean;
  const float* rstd;
  const void* w;
  void* dx;
  float* part;  // [2][blocks][n]: the blocks' sums of dy z and of dy
  int64_t lddy, ldx, ldc, lds, lddx, rows, n;
  bool vdy, vx, vw, vdx;
};

// The saved row's columns c .. c + 7: x itself, or its 8-bit values.
template <typename TX>
__device__ __forceinline__ void saved8(const BwdArgs& a, int64_t row, int64_t c, float (&v)[8]) {
  if (a.x) {
    load8((const TX*)a.x + row * a.ldx, c, a.n, a.vx, v);
  } else if (c < a.n) {
    q8::values8(*reinterpret_cast<const uint2*>(a.codes + row * a.ldc + c),
                q8::scale_of(a.scales[row * a.lds + c / q8::GROUP]), v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
  }
}

template <typename TW>
__device__ __forceinline__ void weight8(const BwdArgs& a, int64_t c, float (&w)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = 1.f;
  if (a.w) load8((const TW*)a.w, c, a.n, a.vw, w);
}

// Teams walk the rows team, team + teams, ...; a thread keeps the sums of its own
// columns over them.  With warp teams the block's warps add theirs in shared memory, in order.
template <typename TX, typename TY, typename TW, int TEAM, int NCH, int BLOCK>
__global__ void __launch_bounds__(BLOCK) backward_kernel(BwdArgs a) {
  __shared__ float2 buf[2][32];
  constexpr int TPB = BLOCK / TEAM;
  const int t = TEAM == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const int64_t team = (int64_t)blockIdx.x * TPB + (TEAM == 32 ? (threadIdx.x >> 5) : 0);
  const float inv_n = 1.f / (float)a.n;
  float sw[NCH][8], sb[NCH][8];
#pragma unroll
  for (int k = 0; k < NCH; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) sw[k][i] = sb[k][i] = 0.f;
  int par = 0;
  for (int64_t row = team; row < a.rows; row += (int64_t)gridDim.x * TPB, par ^= 1) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float g[NCH][8], z[NCH][8];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int64_t c = (int64_t)(t + k * TEAM) * 8;
      load8((const TY*)a.dy + row * a.lddy, c, a.n, a.vdy, g[k]);
      saved8<TX>(a, row, c, z[k]);
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int64_t c = (int64_t)(t + k * TEAM) * 8;
      float w[8];
      weight8<TW>(a, c, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (c + i >= a.n) continue;  // g is 0 there, z would not be
        z[k][i] = (z[k][i] - mean) * rstd;
        sw[k][i] = fmaf(g[k][i], z[k][i], sw[k][i]);
        sb[k][i] += g[k][i];
        g[k][i] *= w[i];
        s.x += g[k][i];
        s.y = fmaf(g[k][i], z[k][i], s.y);
      }
    }
    s = team_sum2<TEAM>(s, buf[par]);
    const float c1 = s.x * inv_n, c2 = s.y * inv_n;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int64_t c = (int64_t)(t + k * TEAM) * 8;
      if (c >= a.n) continue;
      float o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = rstd * (g[k][i] - c1 - z[k][i] * c2);
      store8((TX*)a.dx + row * a.lddx, c, a.n, a.vdx, o);
    }
  }
  if (!a.part) return;
  float* pw = a.part + (int64_t)blockIdx.x * a.n;
  float* pb = pw + (int64_t)gridDim.x * a.n;
  if (TEAM == 32) {
    __shared__ float sum[NCH * 256 + 1];
    for (int which = 0; which < 2; ++which) {
      for (int wp = 0; wp < TPB; ++wp) {
        __syncthreads();
        if ((threadIdx.x >> 5) != wp) continue;
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int c = (t + k * 32) * 8 + i;
            const float v = which ? sb[k][i] : sw[k][i];
            sum[c] = wp == 0 ? v : sum[c] + v;
          }
      }
      __syncthreads();
      for (int c = threadIdx.x; c < a.n; c += BLOCK) (which ? pb : pw)[c] = sum[c];
    }
  } else {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int64_t c = (int64_t)(t + k * TEAM) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < a.n) {
          pw[c + i] = sw[k][i];
          pb[c + i] = sb[k][i];
        }
    }
  }
}

// Rows too wide for registers: dx by a block that walks its row twice ...
template <typename TX, typename TY, typename TW, int BLOCK>
__global__ void __launch_bounds__(BLOCK) backward_long_kernel(BwdArgs a) {
  __shared__ float2 buf[32];
  const int64_t row = blockIdx.x;
  const float mean = a.mean[row], rstd = a.rstd[row];
  const TY* dy = (const TY*)a.dy + row * a.lddy;
  TX* dx = (TX*)a.dx + row * a.lddx;
  float g[8], z[8], w[8];
  float2 s = make_float2(0.f, 0.f);
  for (int64_t c = (int64_t)threadIdx.x * 8; c < a.n; c += BLOCK * 8) {
    load8(dy, c, a.n, a.vdy, g);
    saved8<TX>(a, row, c, z);
    weight8<TW>(a, c, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (c + i >= a.n) continue;
      const float gw = g[i] * w[i];
      s.x += gw;
      s.y = fmaf(gw, (z[i] - mean) * rstd, s.y);
    }
  }
  s = team_sum2<BLOCK>(s, buf);
  const float inv_n = 1.f / (float)a.n, c1 = s.x * inv_n, c2 = s.y * inv_n;
  for (int64_t c = (int64_t)threadIdx.x * 8; c < a.n; c += BLOCK * 8) {
    load8(dy, c, a.n, a.vdy, g);
    saved8<TX>(a, row, c, z);
    weight8<TW>(a, c, w);
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = rstd * (g[i] * w[i] - c1 - (z[i] - mean) * rstd * c2);
    store8(dx, c, a.n, a.vdx, o);
  }
}

// ... and dw, db by blocks of 256 columns (8 a lane) that walk a share of the rows,
// each warp every eighth of them; the warps' sums are added in order.
template <typename TX, typename TY>
__global__ void __launch_bounds__(256) backward_long_sums_kernel(BwdArgs a) {
  __shared__ float sum[2][256];
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 256 + lane * 8;
  float sw[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sb[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int64_t row = (int64_t)blockIdx.y * 8 + wp; row < a.rows; row += (int64_t)gridDim.y * 8) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float g[8], z[8];
    load8((const TY*)a.dy + row * a.lddy, c, a.n, a.vdy, g);
    saved8<TX>(a, row, c, z);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (c + i >= a.n) continue;
      sw[i] = fmaf(g[i], (z[i] - mean) * rstd, sw[i]);
      sb[i] += g[i];
    }
  }
  for (int q = 0; q < 8; ++q) {
    __syncthreads();
    if (q != wp) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sum[0][lane * 8 + i] = q == 0 ? sw[i] : sum[0][lane * 8 + i] + sw[i];
      sum[1][lane * 8 + i] = q == 0 ? sb[i] : sum[1][lane * 8 + i] + sb[i];
    }
  }
  __syncthreads();
  const int64_t cc = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (cc < a.n) {
    a.part[(int64_t)blockIdx.y * a.n + cc] = sum[0][threadIdx.x];
    a.part[((int64_t)gridDim.y + blockIdx.y) * a.n + cc] = sum[1][threadIdx.x];
  }
}

// Widths a team holds: 1024 columns by a warp, 8192 by a block.
constexpr int64_t WARP_MAX = 1024;
constexpr int64_t FWD_MAX = 16384;
constexpr int64_t BWD_MAX = 8192;
constexpr int FWD_WARPS = 4;   // warps a block, warp teams
constexpr int BWD_WARPS = 8;

int bwd_blocks(int64_t rows, int64_t n) {
  if (n > BWD_MAX) return (int)mn<int64_t>(cdiv(rows, 64), 32);
  if (n <= WARP_MAX) return (int)mn<int64_t>(cdiv(rows, BWD_WARPS), 148);
  return (int)mn<int64_t>(rows, 148 * 2);
}

template <typename TX, typename TY, typename TW>
int forward(const FwdArgs& a, cudaStream_t s) {
  if (a.n <= WARP_MAX) {
    const unsigned g = (unsigned)cdiv(a.rows, FWD_WARPS);
    constexpr int B = 32 * FWD_WARPS;
    if (a.n <= 256) forward_kernel<TX, TY, TW, 32, 1, B><<<g, B, 0, s>>>(a);
    else if (a.n <= 512) forward_kernel<TX, TY, TW, 32, 2, B><<<g, B, 0, s>>>(a);
    else if (a.n <= 768) forward_kernel<TX, TY, TW, 32, 3, B><<<g, B, 0, s>>>(a);
    else forward_kernel<TX, TY, TW, 32, 4, B><<<g, B, 0, s>>>(a);
  } else if (a.n <= FWD_MAX) {
    const unsigned g = (unsigned)a.rows;
    if (a.n <= 2048) forward_kernel<TX, TY, TW, 256, 1, 256><<<g, 256, 0, s>>>(a);
    else if (a.n <= 4096) forward_kernel<TX, TY, TW, 256, 2, 256><<<g, 256, 0, s>>>(a);
    else if (a.n <= 8192) forward_kernel<TX, TY, TW, 512, 2, 512><<<g, 512, 0, s>>>(a);
    else forward_kernel<TX, TY, TW, 512, 4, 512><<<g, 512, 0, s>>>(a);
  } else {
    forward_long_kernel<TX, TY, TW, 512><<<(unsigned)a.rows, 512, 0, s>>>(a);
  }
  IFK_CUDA_TRY(cudaGetLastError());
  return IFK_OK;
}

template <typename TX, typename TY, typename TW>
int backward(const BwdArgs& a, cudaStream_t s) {
  const int blocks = bwd_blocks(a.rows, a.n);
  if (a.n <= WARP_MAX) {
    constexpr int B = 32 * BWD_WARPS;
    if (a.n <= 256) backward_kernel<TX, TY, TW, 32, 1, B><<<blocks, B, 0, s>>>(a);
    else if (a.n <= 512) backward_kernel<TX, TY, TW, 32, 2, B><<<blocks, B, 0, s>>>(a);
    else if (a.n <= 768) backward_kernel<TX, TY, TW, 32, 3, B><<<blocks, B, 0, s>>>(a);
    else backward_kernel<TX, TY, TW, 32, 4, B><<<blocks, B, 0, s>>>(a);
  } else if (a.n <= BWD_MAX) {
    if (a.n <= 2048) backward_kernel<TX, TY, TW, 256, 1, 256><<<blocks, 256, 0, s>>>(a);
    else if (a.n <= 4096) backward_kernel<TX, TY, TW, 256, 2, 256><<<blocks, 256, 0, s>>>(a);
    else backward_kernel<TX, TY, TW, 512, 2, 512><<<blocks, 512, 0, s>>>(a);
  } else {
    backward_long_kernel<TX, TY, TW, 512><<<(unsigned)a.rows, 512, 0, s>>>(a);
    if (a.part)
      backward_long_sums_kernel<TX, TY><<<dim3((unsigned)cdiv(a.n, 256), (unsigned)blocks), 256, 0, s>>>(a);
  }
  IFK_CUDA_TRY(cudaGetLastError());
  return IFK_OK;
}

// out[c] = sum over p of part[p][c] in a fixed order: 8 threads a column take every
// eighth p, then one adds the 8.
__global__ void __launch_bounds__(256) sum_parts_kernel(const float* part, int64_t parts, int64_t n, float* out,
                                                        const float* part2, float* out2, int accumulate) {
  __shared__ float sh[8][33];
  const float* src = blockIdx.y ? part2 : part;
  float* dst = blockIdx.y ? out2 : out;
  if (!dst) return;
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  if (c < n)
    for (int64_t p = threadIdx.y; p < parts; p += 8) v += src[p * n + c];
  sh[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0 && c < n) {
    float r = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) r += sh[q][threadIdx.x];
    dst[c] = accumulate ? dst[c] + r : r;
  }
}

}  // namespace

int sum_parts_run(const float* part, int64_t parts, int64_t n, float* out, const float* part2, float* out2,
                  int accumulate, cudaStream_t s) {
  const dim3 grid((unsigned)cdiv(n, 32), part2 ? 2 : 1);
  sum_parts_kernel<<<grid, dim3(32, 8), 0, s>>>(part, parts, n, out, part2, out2, accumulate);
  IFK_CUDA_TRY(cudaGetLastError());
  return IFK_OK;
}

int layernorm_run(const void* x, int64_t ldx, int x_dtype, const void* w, const void* b, int w_dtype, int64_t rows,
                  int64_t n, double eps, void* y, int64_t ldy, int y_dtype, float* mean, float* rstd, int8_t* codes,
                  int64_t ldc, uint8_t* scales, int64_t lds, cudaStream_t s) {
  FwdArgs a;
  a.x = x; a.w = w; a.b = b; a.y = y; a.mean = mean; a.rstd = rstd; a.codes = codes; a.scales = scales;
  a.ldx = ldx; a.ldy = ldy; a.ldc = ldc; a.lds = lds; a.rows = rows; a.n = n; a.eps = (float)eps;
  const bool xf = x_dtype == IFK_F32, yf = y_dtype == IFK_F32, wf = w_dtype == IFK_F32;
  a.vx = xf ? rows_aligned((const float*)x, ldx) : rows_aligned((const __nv_bfloat16*)x, ldx);
  a.vy = yf ? rows_aligned((const float*)y, ldy) : rows_aligned((const __nv_bfloat16*)y, ldy);
  a.vw = ((((uintptr_t)w) | ((uintptr_t)b)) & 15) == 0;
  using B = __nv_bfloat16;
  if (wf) {
    if (xf) return yf ? forward<float, float, float>(a, s) : forward<float, B, float>(a, s);
    return yf ? forward<B, float, float>(a, s) : forward<B, B, float>(a, s);
  }
  if (xf) return yf ? forward<float, float, B>(a, s) : forward<float, B, B>(a, s);
  return yf ? forward<B, float, B>(a, s) : forward<B, B, B>(a, s);
}

size_t layernorm_backward_bytes(int64_t rows, int64_t n) {
  return (size_t)mx<int64_t>(bwd_blocks(rows, n), 1) * (size_t)n * 2 * sizeof(float);
}

int layernorm_backward_run(const void* dy, int64_t lddy, int y_dtype, const void* x, int64_t ldx, int x_dtype,
                           const int8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, const float* mean,
                           const float* rstd, const void* w, int w_dtype, int64_t rows, int64_t n, void* dx,
                           int64_t lddx, float* dw, float* db, float* part, cudaStream_t s) {
  BwdArgs a;
  a.dy = dy; a.x = x; a.codes = codes; a.scales = scales; a.mean = mean; a.rstd = rstd; a.w = w; a.dx = dx;
  a.part = (dw || db) ? part : nullptr;
  a.lddy = lddy; a.ldx = ldx; a.ldc = ldc; a.lds = lds; a.lddx = lddx; a.rows = rows; a.n = n;
  const bool xf = x_dtype == IFK_F32, yf = y_dtype == IFK_F32, wf = w_dtype == IFK_F32;
  a.vdy = yf ? rows_aligned((const float*)dy, lddy) : rows_aligned((const __nv_bfloat16*)dy, lddy);
  a.vx = x && (xf ? rows_aligned((const float*)x, ldx) : rows_aligned((const __nv_bfloat16*)x, ldx));
  a.vdx = xf ? rows_aligned((const float*)dx, lddx) : rows_aligned((const __nv_bfloat16*)dx, lddx);
  a.vw = (((uintptr_t)w) & 15) == 0;
  using B = __nv_bfloat16;
  int rc;
  if (wf) {
    if (xf) rc = yf ? backward<float, float, float>(a, s) : backward<float, B, float>(a, s);
    else rc = yf ? backward<B, float, float>(a, s) : backward<B, B, float>(a, s);
  } else {
    if (xf) rc = yf ? backward<float, float, B>(a, s) : backward<float, B, B>(a, s);
    else rc = yf ? backward<B, float, B>(a, s) : backward<B, B, B>(a, s);
  }
  if (rc != IFK_OK || !a.part) return rc;
  const int64_t parts = bwd_blocks(rows, n);
  return sum_parts_run(part, parts, n, dw, part + parts * n, db, 0, s);
}

}  // namespace ifk
