// Layer norm, backward (ifk_layernorm_backward): dx, and the sums over the rows dw, db.
//
// Bound by memory: dy and the saved rows (as they were, or in 8 bits) are read once, dx
// is written once.  A team of W warps holds a row, COLS columns a lane; the teams of a
// persistent block walk the rows, each lane with the sums of its own columns for dw and
// db in registers, and a ring of rows in shared memory a team, that bulk copies keep
// filled.  At the end the block adds its teams' sums in shared memory and writes one row
// of partial sums; a second kernel adds the blocks'.  The order of every sum is fixed by
// the sizes.  The weight is in shared memory, too: beside the ring there is little L1 left, and
// from L2 it took a third of a row's time.  fp32 arithmetic goes two to an instruction
// (F2): the instructions, not the memory, bound a row of 768 columns in 8 bits otherwise.
// Measured: 16384 x 4096 bf16 from the saved input 73 us (5.5 TB/s) and 3.5 us for the
// blocks' sums, from 8 bits 85 us in all; 65536 x 768 fp32 in 8 bits 80 us (4.4 TB/s).
#include <algorithm>
#include <cstring>

#include "rowvec.cuh"
#include "ifk_internal.h"
#include "pipe.cuh"

namespace ifk {

namespace {

// Bytes of the weight's copy in shared memory (whole blocks of 256 columns).
__host__ __device__ inline size_t weight_bytes(int n) { return (size_t)cdiv(n, 256) * 256 * sizeof(float); }

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
  float* dw;    // where the sums go if one block has them all
  float* db;
  int64_t lddy, ldx, ldc, lds, lddx, rows;
  int n;
  bool w_bf16;
  int W, teams, depth;  // warps a row, teams a block, rows of a team's ring
  int* status;
  bool withhold;  // tests only (IFK_DEBUG_WITHHOLD): the first team's first row never counts as landed
};

constexpr int COLS = 16;         // columns a lane holds: 32 left too few warps for the registers (120 against 80 us
                                 // for 65536 rows of 768 columns in 8 bits)
constexpr int MAX_W = 16;        // warps a row: up to 32 * 16 * 16 = 8192 columns
constexpr int BLOCK_WARPS = 16;  // 128 registers a thread

// The block's sums over its rows: the teams' go to shared memory (2 n floats a team, free by now) and are added
// in order.
template <int V, int NV>
__device__ __forceinline__ void write_sums(const BwdArgs& a, int team, int c0, int step, const float (&sw)[NV][V],
                                           const float (&sb)[NV][V], float* sums) {
  float* mine = sums + (size_t)team * 2 * a.n;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = c0 + k * step + i;
      if (c >= a.n) continue;
      mine[c] = sw[k][i];
      mine[a.n + c] = sb[k][i];
    }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * a.n; c += blockDim.x) {
    float v = sums[c];
    for (int q = 1; q < a.teams; ++q) v += sums[(size_t)q * 2 * a.n + c];
    const int which = c >= a.n, col = c - which * a.n;
    float* out = a.part + ((int64_t)which * gridDim.x + blockIdx.x) * a.n;
    if (gridDim.x == 1) out = which ? a.db : a.dw;
    if (out) out[col] = v;
  }
}
size_t sums_bytes(const BwdArgs& a) { return a.part ? (size_t)a.teams * 2 * a.n * sizeof(float) : 0; }

// The values of a row that a thread works on: dy, and the saved row normalised; 0 past the end.
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

// Rows straight from memory: any alignment and width.
template <typename TX, typename TY, int V, bool Q8>
__global__ void __launch_bounds__(32 * BLOCK_WARPS, 1) backward_kernel(const BwdArgs a) {
  constexpr int NV = COLS / V;
  __shared__ float2 buf[2][BLOCK_WARPS];
  extern __shared__ float sums[];
  const int W = a.W, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, team = warp / W;
  const int c0 = ((warp - team * W) * 32 + lane) * V, step = 32 * W * V;
  const float inv_n = 1.f / (float)a.n;
  const int64_t stride = (int64_t)gridDim.x * a.teams;
  float sw[NV][V], sb[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) sw[k][i] = sb[k][i] = 0.f;
  int par = 0;
  for (int64_t row = (int64_t)blockIdx.x * a.teams + team; row < a.rows; row += stride, par ^= 1) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float g[NV][V], z[NV][V];
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < NV; ++k) row_part<TX, TY, V, Q8>(a, row, c0 + k * step, mean, rstd, g[k], z[k]);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * step;
      float w[V];
      load_param<V>(a.w, a.w_bf16, 1.f, c, a.n, w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        sw[k][i] = fmaf(g[k][i], z[k][i], sw[k][i]);
        sb[k][i] += g[k][i];
        g[k][i] = c + i < a.n ? g[k][i] * w[i] : 0.f;
        s.x += g[k][i];
        s.y = fmaf(g[k][i], z[k][i], s.y);
      }
    }
    s.x = warp_sum(s.x);
    s.y = warp_sum(s.y);
    if (W > 1) {
      // two buffers in turn: the barrier of the next row stands between its writes and these reads
      if (lane == 0) buf[par][warp] = s;
      named_barrier(team + 1, W * 32);
      s = make_float2(0.f, 0.f);
      for (int i = 0; i < W; ++i) {
        const float2 q = buf[par][team * W + i];
        s.x += q.x;
        s.y += q.y;
      }
    }
    const float m1 = s.x * inv_n * rstd, m2 = s.y * inv_n * rstd;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * step;
      if (c >= a.n) continue;
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = fmaf(rstd, g[k][i], fmaf(-m2, z[k][i], -m1));
      store_vec<V>((TX*)a.dx + row * a.lddx, c, a.n, o);
    }
  }
  if (a.part) write_sums<V, NV>(a, team, c0, step, sw, sb, sums);
}

// Where a row's column c stands in the weight's copy in shared memory: the halves of 8 columns a lane
// apart, so that a warp's 16-byte reads are contiguous.
template <int V>
__device__ __forceinline__ int weight_at(int c) {
  return V == 8 ? (c & ~255) + (c & 4) * 32 + ((c >> 1) & 124) + (c & 3) : c;
}

// Rows by bulk copies.  n is a multiple of V, rows of dy and of the saved form are multiples of 16 bytes.
// Once a wait has given up no leader of the block fetches another row: the barrier's phase is still open, and
// arming it again would be one arrival too many.  The block goes on to its end, since its warps meet at
// barriers, with NaN as the weight's first value: each row's sums read it, and all of dx its sums.  Its own sums become
// NaN at the end.
// WARPS: the warps of a row, known when compiled (the columns' addresses are then constants), or 0.
template <typename TX, typename TY, int V, int WARPS, bool Q8>
__global__ void __launch_bounds__(32 * BLOCK_WARPS, 1) backward_ring_kernel(const BwdArgs a) {
  constexpr int NV = COLS / V, H = V / 2;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 buf[2][BLOCK_WARPS];
  __shared__ int failed;
  const int W = WARPS ? WARPS : a.W, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, team = warp / W;
  const int c0 = ((warp - team * W) * 32 + lane) * V, step = 32 * W * V;
  const bool leader = lane == 0 && warp == team * W;
  const int dy_bytes = a.n * (int)sizeof(TY);
  const int x_bytes = Q8 ? (int)q8::pitch(a.n) : a.n * (int)sizeof(TX), bytes = dy_bytes + x_bytes;
  float* weight = reinterpret_cast<float*>(smem);
  uint8_t* rings = smem + weight_bytes(a.n);
  uint8_t* ring = rings + (size_t)team * a.depth * bytes;
  const uint32_t data = (uint32_t)__cvta_generic_to_shared(ring);
  const uint32_t full = (uint32_t)__cvta_generic_to_shared(rings + (size_t)a.teams * a.depth * bytes) +
                        (uint32_t)(team * a.depth * 8);
  const int64_t stride = (int64_t)gridDim.x * a.teams, first = (int64_t)blockIdx.x * a.teams + team;
  if (threadIdx.x == 0) failed = 0;
  if (leader) {
    const int extra = a.withhold && blockIdx.x == 0 && team == 0;
    for (int i = 0; i < a.depth; ++i)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(full + 8 * i), "r"(i == 0 ? 1 + extra : 1)
                   : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  for (int c = threadIdx.x; c < a.n; c += blockDim.x) {
    float w = 1.f;
    if (a.w) w = a.w_bf16 ? __bfloat162float(((const __nv_bfloat16*)a.w)[c]) : ((const float*)a.w)[c];
    weight[weight_at<V>(c)] = w;
  }
  __syncthreads();
  auto fetch = [&](int64_t row, int slot) {
    const uint32_t bar = full + 8 * slot, dst = data + slot * bytes;
    expect(bar, bytes);
    bulk_load(dst, (const TY*)a.dy + row * a.lddy, dy_bytes, bar);
    if (Q8) bulk_load(dst + dy_bytes, a.codes + row * a.ldc, x_bytes, bar);
    else bulk_load(dst + dy_bytes, (const TX*)a.x + row * a.ldx, x_bytes, bar);
  };
  if (leader)
    for (int i = 0; i < a.depth && first + i * stride < a.rows; ++i) fetch(first + i * stride, i);
  const float inv_n = 1.f / (float)a.n;
  F2 sw[NV][H], sb[NV][H];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int i = 0; i < H; ++i) sw[k][i] = sb[k][i] = f2(0.f);
  // what is not in the ring, a row ahead: the statistics, and the scales of the 8-bit rows
  float mean = 0.f, rstd = 0.f;
  uint8_t sc[Q8 ? NV : 1];
  auto ahead = [&](int64_t row) {
    mean = a.mean[row];
    rstd = a.rstd[row];
    if (Q8) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        sc[k % (Q8 ? NV : 1)] = c0 + k * step < a.n ? a.scales[row * a.lds + (c0 + k * step) / q8::GROUP] : 0;
    }
  };
  if (first < a.rows) ahead(first);
  int slot = 0, ph = 0, par = 0;
  for (int64_t row = first; row < a.rows; row += stride, par ^= 1) {
    const float mu = mean, rs = rstd;
    uint8_t s8[Q8 ? NV : 1];
#pragma unroll
    for (int k = 0; k < (Q8 ? NV : 1); ++k) s8[k] = sc[k];
    if (row + stride < a.rows) ahead(row + stride);
    if (!wait_bar(full + 8 * slot, ph, &failed)) *weight = __int_as_float(0x7fffffff);
    const uint8_t* in = ring + (size_t)slot * bytes;
    F2 g[NV][H], z[NV][H], sx = f2(0.f), sy = f2(0.f);
    const F2 nmu = f2(-mu), rs2 = f2(rs);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * step;
      if (c >= a.n) continue;
      float v[V];
      unpack(shared_raw<TY, V>(in, c, a.n), v);
      pairs(v, g[k]);
      if constexpr (Q8) {
        q8::values2<V>(q8::load_codes<V>((const int8_t*)in + dy_bytes + c), q8::scale_of(s8[k]), z[k]);
      } else {
        unpack(shared_raw<TX, V>(in + dy_bytes, c, a.n), v);
        pairs(v, z[k]);
      }
      F2 w[H];
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const float4 q = *reinterpret_cast<const float4*>(weight + weight_at<V>(c + j));
        w[j / 2] = f2(q.x, q.y);
        w[j / 2 + 1] = f2(q.z, q.w);
      }
#pragma unroll
      for (int i = 0; i < H; ++i) {
        z[k][i] = mul(add(z[k][i], nmu), rs2);
        sw[k][i] = fma2(g[k][i], z[k][i], sw[k][i]);
        sb[k][i] = add(sb[k][i], g[k][i]);
        g[k][i] = mul(g[k][i], w[i]);
        sx = add(sx, g[k][i]);
        sy = fma2(g[k][i], z[k][i], sy);
      }
    }
    float2 s = make_float2(warp_sum(sum(sx)), warp_sum(sum(sy)));
    if (W > 1) {
      // two buffers in turn: the barrier of the next row stands between its writes and these reads
      if (lane == 0) buf[par][warp] = s;
      named_barrier(team + 1, W * 32);
      s = make_float2(0.f, 0.f);
      for (int i = 0; i < W; ++i) {
        const float2 q = buf[par][team * W + i];
        s.x += q.x;
        s.y += q.y;
      }
    }
    // every lane of the team has read the row
    if (leader && row + a.depth * stride < a.rows && !*(volatile int*)&failed)
      fetch(row + a.depth * stride, slot);
    if (++slot == a.depth) {
      slot = 0;
      ph ^= 1;
    }
    const F2 m1 = f2(-s.x * inv_n * rs), m2 = f2(-s.y * inv_n * rs);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = c0 + k * step;
      if (c >= a.n) continue;
      F2 q[H];
      float o[V];
#pragma unroll
      for (int i = 0; i < H; ++i) q[i] = fma2(rs2, g[k][i], fma2(m2, z[k][i], m1));
      singles(q, o);
      store_vec<V, true>((TX*)a.dx + row * a.lddx, c, a.n, o);
    }
  }
  __syncthreads();
  const bool bad = failed;
  const float nan = __int_as_float(0x7fffffff);
  if (bad) {
    if (threadIdx.x == 0) {
      linger();
      if (a.status) *a.status = IFK_ERR_TIMEOUT;
    }
    __syncthreads();
  }
  if (a.part) {
    float w[NV][V], b[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      singles(sw[k], w[k]);
      singles(sb[k], b[k]);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (bad) w[k][i] = b[k][i] = nan;
    }
    write_sums<V, NV>(a, team, c0, step, w, b, reinterpret_cast<float*>(smem));
  }
}

// Rows too wide for registers: dx by a block that walks its row twice ...
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

// Persistent blocks: one an SM, fewer when the rows do not fill them (a block's partial sums are written
// and read once).  The number of blocks depends on the sizes alone: it is the number of partial sums.
int row_warps(int64_t n) {
  const int w = (int)cdiv(n, 32 * COLS);
  return w == 5 ? 6 : w == 7 ? 8 : w;  // the counts that have a kernel of their own
}
int block_teams(int64_t n) { return std::max(1, BLOCK_WARPS / row_warps(n)); }
int64_t parts_of(int64_t rows, int64_t n) {
  if (row_warps(n) > MAX_W) return std::min<int64_t>(cdiv(rows, 64), 32);
  return std::min<int64_t>(cdiv(rows, block_teams(n)), 148);
}

constexpr size_t RING_BYTES = 200 * 1024;

// Whether the rows can come by bulk copies; sets the ring's depth.
template <typename TX, typename TY, int V, bool Q8>
bool ring_ok(BwdArgs& a, size_t* row) {
  const size_t dy = (size_t)a.n * sizeof(TY), x = Q8 ? (size_t)q8::pitch(a.n) : (size_t)a.n * sizeof(TX);
  *row = dy + x;
  a.depth = (int)std::min<size_t>(8, (RING_BYTES - weight_bytes(a.n)) / (a.teams * *row));
  return V > 1 && a.n % V == 0 && a.depth >= 2 && dy % 16 == 0 && x % 16 == 0 &&
         rows_allow<uint8_t>(a.dy, a.lddy * (int64_t)sizeof(TY), 16) &&
         (Q8 || rows_allow<uint8_t>(a.x, a.ldx * (int64_t)sizeof(TX), 16));
}

template <typename K>
int launch(K kernel, int* done_dev, unsigned blocks, unsigned threads, size_t smem, const BwdArgs& a, cudaStream_t s) {
  int dev = 0;
  IFK_CUDA_TRY(cudaGetDevice(&dev));
  if (*done_dev != dev) {
    IFK_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)RING_BYTES + 2048));
    *done_dev = dev;
  }
  kernel<<<blocks, threads, smem, s>>>(a);
  IFK_CUDA_TRY(cudaGetLastError());
  return IFK_OK;
}

template <typename TX, typename TY, int V, int WARPS, bool Q8>
int launch_ring(const BwdArgs& a, unsigned blocks, size_t row, cudaStream_t s) {
  static thread_local int done_dev = -1;
  return launch(backward_ring_kernel<TX, TY, V, WARPS, Q8>, &done_dev, blocks, 32 * a.W * a.teams,
                std::max<size_t>(weight_bytes(a.n) + a.teams * a.depth * (row + 8), sums_bytes(a)), a, s);
}

template <typename TX, typename TY, int V, bool Q8>
int backward(BwdArgs& a, cudaStream_t s) {
  const unsigned parts = (unsigned)parts_of(a.rows, a.n);
  a.W = row_warps(a.n);
  if (a.W > MAX_W) {
    backward_long_kernel<TX, TY, V, Q8><<<(unsigned)a.rows, 512, 0, s>>>(a);
    if (a.part)
      backward_long_sums_kernel<TX, TY, V, Q8><<<dim3((unsigned)cdiv(a.n, 32 * V), parts), 256, 0, s>>>(a);
    IFK_CUDA_TRY(cudaGetLastError());
    return IFK_OK;
  }
  a.teams = block_teams(a.n);
  if constexpr (V > 1) {
    size_t row;
    if (ring_ok<TX, TY, V, Q8>(a, &row)) {
      switch (a.W) {
        case 1: return launch_ring<TX, TY, V, 1, Q8>(a, parts, row, s);
        case 2: return launch_ring<TX, TY, V, 2, Q8>(a, parts, row, s);
        case 3: return launch_ring<TX, TY, V, 3, Q8>(a, parts, row, s);
        case 4: return launch_ring<TX, TY, V, 4, Q8>(a, parts, row, s);
        case 6: return launch_ring<TX, TY, V, 6, Q8>(a, parts, row, s);
        case 8: return launch_ring<TX, TY, V, 8, Q8>(a, parts, row, s);
        default: return launch_ring<TX, TY, V, 0, Q8>(a, parts, row, s);
      }
    }
  }
  static thread_local int done_dev = -1;
  return launch(backward_kernel<TX, TY, V, Q8>, &done_dev, parts, 32 * a.W * a.teams, sums_bytes(a), a, s);
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
                                                         const float* part2, float* out2) {
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
  if (threadIdx.x == 0 && o < n) dst[o] = v;
}

}  // namespace

size_t layernorm_backward_bytes(int64_t rows, int64_t n) {
  return (size_t)std::max<int64_t>(parts_of(rows, n), 1) * (size_t)n * 2 * sizeof(float);
}

int layernorm_backward_run(const void* dy, int64_t lddy, int y_dtype, const void* x, int64_t ldx, int x_dtype,
                           const int8_t* codes, int64_t ldc, const uint8_t* scales, int64_t lds, const float* mean,
                           const float* rstd, const void* w, int w_dtype, int64_t rows, int64_t n, void* dx,
                           int64_t lddx, float* dw, float* db, float* part, int* status, bool withhold,
                           cudaStream_t s) {
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
  a.dw = dw;
  a.db = db;
  a.lddy = lddy;
  a.ldx = ldx;
  a.ldc = ldc;
  a.lds = lds;
  a.lddx = lddx;
  a.rows = rows;
  a.n = (int)n;
  a.w_bf16 = w_dtype == IFK_BF16;
  a.teams = a.depth = 1;
  a.status = status;
  a.withhold = withhold;
  using B = __nv_bfloat16;
  int rc;
  if (x_dtype == IFK_F32) rc = y_dtype == IFK_F32 ? backward_any<float, float>(a, s) : backward_any<float, B>(a, s);
  else rc = y_dtype == IFK_F32 ? backward_any<B, float>(a, s) : backward_any<B, B>(a, s);
  if (rc != IFK_OK || !a.part) return rc;
  const int64_t parts = parts_of(rows, n);
  if (parts == 1 && row_warps(n) <= MAX_W) return IFK_OK;  // the one block has written them
  sum_parts_kernel<<<dim3((unsigned)cdiv(n, 32), 2), dim3(32, 32), 0, s>>>(part, parts, n, dw, part + parts * n, db);
  IFK_CUDA_TRY(cudaGetLastError());
  return IFK_OK;
}

}  // namespace ifk
