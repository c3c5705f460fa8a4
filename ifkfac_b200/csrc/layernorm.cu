// Layer norm, forward (ifk_layernorm).
//
// One pass bound by memory: x is read once into registers (as it is in memory, so a
// bf16 row takes half of them), the statistics are two sums over the registers, and y
// (and the 8-bit rows of x) are written.  A team of W warps holds a row, four neighbouring
// columns a lane at a time, or one where a row is not aligned for that; a lane holds up to
// 32.  Four, also where eight bf16 are one 16-byte access: a warp's reads of the fp32
// weight and bias are then contiguous, and they, from L1, are most of what the load unit
// does (16384 x 4096 bf16: 51 us against 58; with 8-bit rows, where eight halve the
// groups' shuffles, 76 against 70, but the sums' order, and so y, would depend on whether
// the rows are kept).  A row no wider than one warp holds needs no barrier.  Measured:
// 32768 x 1280 fp32 to bf16 41 us (6.1 TB/s), 16384 x 4096 bf16 51 us (5.3 TB/s),
// 65536 x 768 fp32 to bf16 with 8-bit rows 62 us (5.7 TB/s).
#include <algorithm>
#include <cstring>

#include "rowvec.cuh"
#include "ifk_internal.h"

namespace ifk {

namespace {

struct FwdArgs {
  const void* x;
  const void* w;
  const void* b;
  void* y;
  float* mean;
  float* rstd;
  int8_t* codes;
  uint8_t* scales;
  int64_t ldx, ldy, ldc, lds, rows;
  int n, pitch;
  float eps;
  bool w_bf16;
  int W;  // warps a row
};

constexpr int ROWS_PER_BLOCK = 4;  // of one warp each

// Sums over the W warps of a row; buf is used once.
__device__ __forceinline__ float team_sum(float v, int W, float* buf) {
  v = warp_sum(v);
  if (W == 1) return v;
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = buf[0];
  for (int i = 1; i < W; ++i) r += buf[i];
  return r;
}

// 8-bit rows of x, written as ifk_q8_quantize writes them: a lane's V columns of a group with the maximum m.
template <int V>
__device__ __forceinline__ void write_group(int8_t* codes, uint8_t* scales, int pitch, int c, const float (&v)[V],
                                            uint32_t m) {
  if (c >= pitch) return;
  const uint32_t s = q8::scale_byte(m);
  q8::store_codes<V>(codes + c, v, m, s);
  if ((c & (q8::GROUP - 1)) == 0) scales[c / q8::GROUP] = (uint8_t)s;
}
template <int V>
__device__ __forceinline__ void write_codes(int8_t* codes, uint8_t* scales, int pitch, int c, const float (&v)[V]) {
  write_group<V>(codes, scales, pitch, c, v, q8::group_max_bits<V>(v));
}

// The mean is taken twice: the second sum, over x less the first mean, carries what the
// first one rounded away, and the variance is that of the differences.
struct Stats {
  float m1, c1, rstd;  // mean = m1 + c1
};
__device__ __forceinline__ Stats finish_stats(float m1, float sd, float sd2, float inv_n, float eps) {
  Stats t;
  t.m1 = m1;
  t.c1 = sd * inv_n;
  t.rstd = 1.f / sqrtf(fmaxf(fmaf(-t.c1, t.c1, sd2 * inv_n), 0.f) + eps);
  return t;
}

// PLAIN: n is a multiple of V, w and b are there and fp32.
template <typename TY, int V, bool PLAIN>
__device__ __forceinline__ void write_out(const FwdArgs& a, TY* y, int c, const float (&v)[V], const Stats& t) {
  float w[V], b[V], o[V];
  if constexpr (PLAIN) {
    load_f32<V>((const float*)a.w, c, w);
    load_f32<V>((const float*)a.b, c, b);
    F2 q[V / 2], w2[V / 2], b2[V / 2];
    pairs(v, q);
    pairs(w, w2);
    pairs(b, b2);
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      q[i] = fma2(mul(add(add(q[i], f2(-t.m1)), f2(-t.c1)), f2(t.rstd)), w2[i], b2[i]);
    singles(q, o);
  } else {
    load_param<V>(a.w, a.w_bf16, 1.f, c, a.n, w);
    load_param<V>(a.b, a.w_bf16, 0.f, c, a.n, b);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = fmaf((v[i] - t.m1 - t.c1) * t.rstd, w[i], b[i]);
  }
  store_vec<V, PLAIN>(y, c, a.n, o);
}

// WARPS: the warps of a row, known when compiled (the columns' addresses are then constants), or 0.
template <int WARPS>
constexpr int max_threads() { return WARPS == 0 ? 512 : WARPS == 1 ? 32 * ROWS_PER_BLOCK : 32 * WARPS; }
// 64 registers a thread.
template <int WARPS>
constexpr int min_blocks() { return 1024 / max_threads<WARPS>(); }

template <typename TX, typename TY, int V, int NV, bool PLAIN, int WARPS>
__global__ void __launch_bounds__(max_threads<WARPS>(), min_blocks<WARPS>()) forward_kernel(const FwdArgs a) {
  __shared__ float buf[3][32];
  const int W = WARPS ? WARPS : a.W, lane = threadIdx.x & 31;
  const int64_t row = W == 1 ? (int64_t)blockIdx.x * ROWS_PER_BLOCK + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.rows) return;  // whole warps of one-warp rows
  const int c0 = (W == 1 ? lane : (int)threadIdx.x) * V, step = 32 * W * V;
  const TX* x = (const TX*)a.x + row * a.ldx;
  TY* y = (TY*)a.y + row * a.ldy;
  const float inv_n = 1.f / (float)a.n;
  Raw<TX, V> r[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) r[k] = load_raw<TX, V, PLAIN>(x, c0 + k * step, a.n);
  float s = 0.f, sd = 0.f, sd2 = 0.f;
  if constexpr (PLAIN) {
    F2 s2 = f2(0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float v[V];
      F2 q[V / 2];
      unpack(r[k], v);
      pairs(v, q);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) s2 = add(s2, q[i]);
    }
    s = sum(s2);
  } else {
    // even and odd columns apart, as the pairs of the plain form: the same bits
    float odd = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float v[V];
      unpack(r[k], v);
#pragma unroll
      for (int i = 0; i < V; ++i) (i & 1 ? odd : s) += v[i];
    }
    s += odd;
  }
  const float m1 = team_sum(s, W, buf[0]) * inv_n;
  if constexpr (PLAIN) {
    F2 d1 = f2(0.f), d2 = f2(0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (c0 + k * step >= a.n) continue;
      float v[V];
      F2 q[V / 2];
      unpack(r[k], v);
      pairs(v, q);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const F2 d = add(q[i], f2(-m1));
        d1 = add(d1, d);
        d2 = fma2(d, d, d2);
      }
    }
    sd = sum(d1);
    sd2 = sum(d2);
  } else {
    float odd = 0.f, odd2 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * step;
      float v[V];
      unpack(r[k], v);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = c + i < a.n ? v[i] - m1 : 0.f;
        (i & 1 ? odd : sd) += d;
        float& q = i & 1 ? odd2 : sd2;
        q = fmaf(d, d, q);
      }
    }
    sd += odd;
    sd2 += odd2;
  }
  sd = warp_sum(sd);
  sd2 = warp_sum(sd2);
  if (W > 1) {
    if (lane == 0) {
      buf[1][threadIdx.x >> 5] = sd;
      buf[2][threadIdx.x >> 5] = sd2;
    }
    __syncthreads();
    sd = sd2 = 0.f;
    for (int i = 0; i < W; ++i) {
      sd += buf[1][i];
      sd2 += buf[2][i];
    }
  }
  const Stats t = finish_stats(m1, sd, sd2, inv_n, a.eps);
  if (c0 == 0) {
    if (a.mean) a.mean[row] = t.m1 + t.c1;
    if (a.rstd) a.rstd[row] = t.rstd;
  }
  int8_t* codes = a.codes + row * a.ldc;
  uint8_t* scales = a.scales + row * a.lds;
  if constexpr (NV == 1) {
    float v[V];
    unpack(r[0], v);
    if (a.codes) write_codes<V>(codes, scales, a.pitch, c0, v);
    if (c0 < a.n) write_out<TY, V, PLAIN>(a, y, c0, v, t);
  } else {
    static_assert(NV % 2 == 0, "accesses are handled in pairs");
#pragma unroll
    for (int k = 0; k < NV; k += 2) {
      const int c = c0 + k * step;
      float v[V], u[V];
      unpack(r[k], v);
      unpack(r[k + 1], u);
      if (a.codes) {
        uint32_t mv, mu;
        q8::group_max_bits_of_two<V>(v, u, mv, mu);
        write_group<V>(codes, scales, a.pitch, c, v, mv);
        write_group<V>(codes, scales, a.pitch, c + step, u, mu);
      }
      if (c < a.n) write_out<TY, V, PLAIN>(a, y, c, v, t);
      if (c + step < a.n) write_out<TY, V, PLAIN>(a, y, c + step, u, t);
    }
  }
}

// Rows too wide for registers: a block walks its row three times (from L2 after the first).
template <typename TX, typename TY, int V>
__global__ void __launch_bounds__(512) forward_long_kernel(const FwdArgs a) {
  __shared__ float buf[3][32];
  constexpr int W = 16, step = 32 * W * V;
  const int64_t row = blockIdx.x;
  const int c0 = threadIdx.x * V;
  const TX* x = (const TX*)a.x + row * a.ldx;
  TY* y = (TY*)a.y + row * a.ldy;
  const float inv_n = 1.f / (float)a.n;
  float v[V], s = 0.f, sd = 0.f, sd2 = 0.f;
  for (int c = c0; c < a.n; c += step) {
    unpack(load_raw<TX, V>(x, c, a.n), v);
#pragma unroll
    for (int i = 0; i < V; ++i) s += v[i];
  }
  const float m1 = team_sum(s, W, buf[0]) * inv_n;
  for (int c = c0; c < a.n; c += step) {
    unpack(load_raw<TX, V>(x, c, a.n), v);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = c + i < a.n ? v[i] - m1 : 0.f;
      sd += d;
      sd2 = fmaf(d, d, sd2);
    }
  }
  sd = team_sum(sd, W, buf[1]);
  sd2 = team_sum(sd2, W, buf[2]);
  const Stats t = finish_stats(m1, sd, sd2, inv_n, a.eps);
  if (threadIdx.x == 0) {
    if (a.mean) a.mean[row] = t.m1 + t.c1;
    if (a.rstd) a.rstd[row] = t.rstd;
  }
  // every warp runs its last round whole: the groups' shuffles need each lane
  for (int cw = (threadIdx.x & ~31) * V; cw < a.pitch; cw += step) {
    const int c = cw + (threadIdx.x & 31) * V;
    unpack(load_raw<TX, V>(x, c, a.n), v);
    if (a.codes) write_codes<V>(a.codes + row * a.ldc, a.scales + row * a.lds, a.pitch, c, v);
    if (c < a.n) write_out<TY, V, false>(a, y, c, v, t);
  }
}

template <typename TX, typename TY, int V, int NV, bool PLAIN>
void launch(FwdArgs& a, cudaStream_t s) {
  const unsigned rows = (unsigned)a.rows;
  if (a.W == 1)
    forward_kernel<TX, TY, V, NV, PLAIN, 1>
        <<<(unsigned)cdiv(a.rows, ROWS_PER_BLOCK), 32 * ROWS_PER_BLOCK, 0, s>>>(a);
  else if (PLAIN && a.W == 2)
    forward_kernel<TX, TY, V, NV, PLAIN, PLAIN ? 2 : 0><<<rows, 32 * a.W, 0, s>>>(a);
  else if (PLAIN && a.W == 4)
    forward_kernel<TX, TY, V, NV, PLAIN, PLAIN ? 4 : 0><<<rows, 32 * a.W, 0, s>>>(a);
  else
    forward_kernel<TX, TY, V, NV, PLAIN, 0><<<rows, 32 * a.W, 0, s>>>(a);
}

// Accesses a lane makes of a row: 32 columns' at most; fewer, by more warps a row, while the rows
// alone do not give each SM eight warps.
template <typename TX, typename TY, int V>
int forward(FwdArgs& a, cudaStream_t s) {
  constexpr int MAXV = 32 / V;
  const int acc = a.pitch / V;  // accesses of a row (with the padding of its last group)
  int W = (int)cdiv(acc, 32 * MAXV);
  if (W > 16) {
    forward_long_kernel<TX, TY, V><<<(unsigned)a.rows, 512, 0, s>>>(a);
  } else {
    while (W < 16 && a.rows * W < 148 * 8 && acc > 32 * W) W = std::min(2 * W, 16);
    a.W = W;
    const int nv = (int)cdiv(acc, 32 * W);
    const bool plain = V > 1 && a.n % V == 0 && a.w && a.b && !a.w_bf16;
    if constexpr (V == 1) {
      if (nv <= 4) launch<TX, TY, V, 4, false>(a, s);
      else if (nv <= 8) launch<TX, TY, V, 8, false>(a, s);
      else if (nv <= 16) launch<TX, TY, V, 16, false>(a, s);
      else launch<TX, TY, V, 32, false>(a, s);
    } else if (!plain) {
      if (2 * nv <= MAXV) launch<TX, TY, V, MAXV / 2, false>(a, s);
      else launch<TX, TY, V, MAXV, false>(a, s);
    } else if (nv <= 1) {
      launch<TX, TY, V, 1, true>(a, s);
    } else if (nv <= 2) {
      launch<TX, TY, V, 2, true>(a, s);
    } else if (nv <= 4) {
      launch<TX, TY, V, 4, true>(a, s);
    } else if (nv <= 6) {
      launch<TX, TY, V, 6, true>(a, s);
    } else {
      launch<TX, TY, V, MAXV, true>(a, s);
    }
  }
  IFK_CUDA_TRY(cudaGetLastError());
  return IFK_OK;
}

template <typename TX, typename TY>
int forward_any(FwdArgs& a, cudaStream_t s) {
  const bool four = rows_allow<TX>(a.x, a.ldx, 4) && rows_allow<TY>(a.y, a.ldy, 4) &&
                    ((((uintptr_t)a.w) | ((uintptr_t)a.b)) & 15) == 0;
  return four ? forward<TX, TY, 4>(a, s) : forward<TX, TY, 1>(a, s);
}

}  // namespace

int layernorm_run(const void* x, int64_t ldx, int x_dtype, const void* w, const void* b, int w_dtype, int64_t rows,
                  int64_t n, double eps, void* y, int64_t ldy, int y_dtype, float* mean, float* rstd, int8_t* codes,
                  int64_t ldc, uint8_t* scales, int64_t lds, cudaStream_t s) {
  FwdArgs a;
  a.x = x;
  a.w = w;
  a.b = b;
  a.y = y;
  a.mean = mean;
  a.rstd = rstd;
  a.codes = codes;
  a.scales = scales;
  a.ldx = ldx;
  a.ldy = ldy;
  a.ldc = ldc;
  a.lds = lds;
  a.rows = rows;
  a.n = (int)n;
  a.pitch = (int)q8::pitch(n);
  a.eps = (float)eps;
  a.w_bf16 = w_dtype == IFK_BF16;
  a.W = 1;
  using B = __nv_bfloat16;
  if (x_dtype == IFK_F32) return y_dtype == IFK_F32 ? forward_any<float, float>(a, s) : forward_any<float, B>(a, s);
  return y_dtype == IFK_F32 ? forward_any<B, float>(a, s) : forward_any<B, B>(a, s);
}

}  // namespace ifk
